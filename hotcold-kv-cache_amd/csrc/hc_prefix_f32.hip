// The attention behind a shared prompt, float inputs (kernels in hc_prefix_kernels.h).
#include "hc_prefix_kernels.h"

namespace hc {
template void launch_prefix<float>(const PrefixArgs&, int64_t, hipStream_t);
}
