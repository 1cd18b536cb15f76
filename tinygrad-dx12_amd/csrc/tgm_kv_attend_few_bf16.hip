// kv_attend_few for bf16 queries.
#include "tgm_kv_attend_few.h"

namespace tgm {
template void attend_few<TGM_BF16>(const AttendLaunch&, hipStream_t);
}
