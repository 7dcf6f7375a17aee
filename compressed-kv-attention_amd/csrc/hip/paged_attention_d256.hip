// Attention over a paged cache, channels held as 256 (paged_attention.h).
#include "paged_attention_launch.h"

namespace kvexp_launch {
KVEXP_PAGED_LAUNCH(256)
} // namespace kvexp_launch
