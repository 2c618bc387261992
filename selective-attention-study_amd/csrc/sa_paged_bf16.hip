// Attention over a paged bf16 cache.

#include "sa_paged.h"

namespace sa_host {

int paged_bf16(const PagedLaunch& c) { return paged_entry<PagedBF16>(c); }

}  // namespace sa_host
