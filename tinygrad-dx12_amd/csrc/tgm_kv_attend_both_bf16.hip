// kv_attend_both for bf16 queries.
#include "tgm_kv_attend_both.h"

namespace tgm {
template void attend_both<TGM_BF16>(const AttendLaunch&, const AttendLaunch&, hipStream_t);
}
