// Attention over a paged fp32 cache.

#include "sa_paged.h"

namespace sa_host {

int paged_f32(const PagedLaunch& c) { return paged_entry<PagedF32>(c); }

}  // namespace sa_host
