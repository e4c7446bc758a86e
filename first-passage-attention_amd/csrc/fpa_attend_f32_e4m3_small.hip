// fp32 queries, e4m3 pages, head sizes 16 to 64.
#include "fpa_attend.h"

namespace fpa {
template hipError_t launch_attend_small<float, e4m3>(const AttendParams &, int, hipStream_t);
}
