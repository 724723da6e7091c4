// Attention over a cache in pages, head dims 65 to 128.
#include "attention_paged.h"

namespace th {
int paged_attention_128(const th_paged_desc* d, th_launch** out) { return launch_dim<128>(d, out); }
}  // namespace th
