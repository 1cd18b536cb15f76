// kv_attend_many for bf16 queries.
#include "tgm_kv_attend_many.h"

namespace tgm {
template void attend_many<TGM_BF16>(const AttendLaunch&, hipStream_t);
}
