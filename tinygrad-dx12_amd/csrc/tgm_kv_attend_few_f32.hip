// kv_attend_few for f32 queries.
#include "tgm_kv_attend_few.h"

namespace tgm {
template void attend_few<TGM_F32>(const AttendLaunch&, hipStream_t);
}
