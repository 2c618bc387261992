// The vocabulary loss with bf16 products.

#include "sa_xent.h"

namespace sa_host {

int64_t xent_bytes_bf16(const XentCall& c, bool backward) { return xent_bytes<XBF16>(c, backward); }
int xent_bf16(const XentCall& c, bool backward) { return backward ? xent_backward<XBF16>(c) : xent_forward<XBF16>(c); }

}  // namespace sa_host
