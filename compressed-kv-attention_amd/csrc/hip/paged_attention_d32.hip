// Attention over a paged cache, channels held as 32 (paged_attention.h).
#include "paged_attention_launch.h"

namespace kvexp_launch {
KVEXP_PAGED_LAUNCH(32)
} // namespace kvexp_launch
