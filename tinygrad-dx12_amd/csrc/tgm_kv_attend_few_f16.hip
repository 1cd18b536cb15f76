// kv_attend_few for f16 queries.
#include "tgm_kv_attend_few.h"

namespace tgm {
template void attend_few<TGM_F16>(const AttendLaunch&, hipStream_t);
}
