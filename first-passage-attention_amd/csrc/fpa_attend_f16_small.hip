// fp16 queries, fp16 pages, head sizes 16 to 64.
#include "fpa_attend.h"

namespace fpa {
template hipError_t launch_attend_small<f16, f16>(const AttendParams &, int, hipStream_t);
}
