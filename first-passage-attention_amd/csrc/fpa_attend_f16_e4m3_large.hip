// fp16 queries, e4m3 pages, head sizes 128 and 256.
#include "fpa_attend.h"

namespace fpa {
template hipError_t launch_attend_large<f16, e4m3>(const AttendParams &, int, hipStream_t);
}
