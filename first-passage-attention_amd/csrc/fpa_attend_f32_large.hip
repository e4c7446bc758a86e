// fp32 queries, fp32 pages, head sizes 128 and 256.
#include "fpa_attend.h"

namespace fpa {
template hipError_t launch_attend_large<float, float>(const AttendParams &, int, hipStream_t);
}
