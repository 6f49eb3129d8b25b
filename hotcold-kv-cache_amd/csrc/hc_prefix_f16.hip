// The attention behind a shared prompt, half_t inputs (kernels in hc_prefix_kernels.h).
#include "hc_prefix_kernels.h"

namespace hc {
template void launch_prefix<half_t>(const PrefixArgs&, int64_t, hipStream_t);
}
