// kv_attend_many for f32 queries.
#include "tgm_kv_attend_many.h"

namespace tgm {
template void attend_many<TGM_F32>(const AttendLaunch&, hipStream_t);
}
