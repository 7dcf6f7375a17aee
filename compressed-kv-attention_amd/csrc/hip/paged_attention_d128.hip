// Attention over a paged cache, channels held as 128 (paged_attention.h).
#include "paged_attention_launch.h"

namespace kvexp_launch {
KVEXP_PAGED_LAUNCH(128)
} // namespace kvexp_launch
