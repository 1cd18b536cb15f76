// kv_attend_many for f16 queries.
#include "tgm_kv_attend_many.h"

namespace tgm {
template void attend_many<TGM_F16>(const AttendLaunch&, hipStream_t);
}
