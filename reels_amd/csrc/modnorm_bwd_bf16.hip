#include "modnorm_bwd_impl.h"

namespace reels {
template void launch_mod_bwd<REELS_HIP_BF16>(const ModBwdArgs&, ModForm, bool, bool, int64_t, hipStream_t);
}  // namespace reels
