// Attention over a paged cache, channels held as 192 (paged_attention.h).
#include "paged_attention_launch.h"

namespace kvexp_launch {
KVEXP_PAGED_LAUNCH(192)
} // namespace kvexp_launch
