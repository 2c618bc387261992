// The vocabulary loss with fp32 products.

#include "sa_xent.h"

namespace sa_host {

int64_t xent_bytes_f32(const XentCall& c, bool backward) { return xent_bytes<XF32>(c, backward); }
int xent_f32(const XentCall& c, bool backward) { return backward ? xent_backward<XF32>(c) : xent_forward<XF32>(c); }

}  // namespace sa_host
