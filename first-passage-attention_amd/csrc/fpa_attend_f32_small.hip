// fp32 queries, fp32 pages, head sizes 16 to 64.
#include "fpa_attend.h"

namespace fpa {
template hipError_t launch_attend_small<float, float>(const AttendParams &, int, hipStream_t);
}
