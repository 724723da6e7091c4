// Attention over a cache in pages, head dims 129 to 256.
#include "attention_paged.h"

namespace th {
int paged_attention_256(const th_paged_desc* d, th_launch** out) { return launch_dim<256>(d, out); }
}  // namespace th
