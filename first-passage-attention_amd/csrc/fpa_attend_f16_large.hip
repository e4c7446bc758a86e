// fp16 queries, fp16 pages, head sizes 128 and 256.
#include "fpa_attend.h"

namespace fpa {
template hipError_t launch_attend_large<f16, f16>(const AttendParams &, int, hipStream_t);
}
