// The vocabulary loss with fp16 products.

#include "sa_xent.h"

namespace sa_host {

int64_t xent_bytes_f16(const XentCall& c, bool backward) { return xent_bytes<XF16>(c, backward); }
int xent_f16(const XentCall& c, bool backward) { return backward ? xent_backward<XF16>(c) : xent_forward<XF16>(c); }

}  // namespace sa_host
