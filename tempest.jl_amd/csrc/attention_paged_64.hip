// Attention over a cache in pages, head dims up to 64.
#include "attention_paged.h"

namespace th {
int paged_attention_64(const th_paged_desc* d, th_launch** out) { return launch_dim<64>(d, out); }
}  // namespace th
