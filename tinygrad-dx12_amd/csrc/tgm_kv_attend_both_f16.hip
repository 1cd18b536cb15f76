// kv_attend_both for f16 queries.
#include "tgm_kv_attend_both.h"

namespace tgm {
template void attend_both<TGM_F16>(const AttendLaunch&, const AttendLaunch&, hipStream_t);
}
