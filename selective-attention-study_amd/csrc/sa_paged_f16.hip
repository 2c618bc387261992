// Attention over a paged fp16 cache.

#include "sa_paged.h"

namespace sa_host {

int paged_f16(const PagedLaunch& c) { return paged_entry<PagedF16>(c); }

}  // namespace sa_host
