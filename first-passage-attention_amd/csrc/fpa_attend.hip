// fpa_attend.hip -- how the attention against a cache is cut into parts, and its dispatch over types; the kernels are in
// fpa_attend.h, built by the fpa_attend_*.hip files.
#include "fpa_attend.h"

namespace fpa {

extern template hipError_t launch_attend_small<f16, f16>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_large<f16, f16>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_small<float, float>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_large<float, float>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_small<f16, e4m3>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_large<f16, e4m3>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_small<float, e4m3>(const AttendParams &, int, hipStream_t);
extern template hipError_t launch_attend_large<float, e4m3>(const AttendParams &, int, hipStream_t);

hipError_t launch_attend(const AttendParams &p, int dtype, int store, int D, hipStream_t s) {
    if (dtype == ST_F16 && store == ST_F16) return D <= 64 ? launch_attend_small<f16, f16>(p, D, s) : launch_attend_large<f16, f16>(p, D, s);
    if (dtype == ST_F32 && store == ST_F32) return D <= 64 ? launch_attend_small<float, float>(p, D, s) : launch_attend_large<float, float>(p, D, s);
    if (dtype == ST_F16 && store == ST_E4M3) return D <= 64 ? launch_attend_small<f16, e4m3>(p, D, s) : launch_attend_large<f16, e4m3>(p, D, s);
    if (dtype == ST_F32 && store == ST_E4M3) return D <= 64 ? launch_attend_small<float, e4m3>(p, D, s) : launch_attend_large<float, e4m3>(p, D, s);
    return hipErrorInvalidValue;
}

int attend_waves(int D) { return waves(D); }

int attend_rows(int64_t rows, int D, int dtype) { return CW * prefix_sets(D, rows, dtype == ST_F32); }

#ifndef PARTS_WG
#define PARTS_WG 256
#endif
#ifndef ALONE_PAGES
#define ALONE_PAGES 16
#define ALONE_ITEMS 256
#endif

int attend_steps(int D, int dtype, int store, int64_t N, bool prefix, int sets) {
    const int kind = N > 4 ? 0 : N > 1 || prefix ? 4 : 1;
    if (store == ST_F16) return steps_of<f16, f16>(D, kind, sets);
    if (store == ST_F32) return steps_of<float, float>(D, kind, sets);
    return dtype == ST_F16 ? steps_of<f16, e4m3>(D, kind, sets) : steps_of<float, e4m3>(D, kind, sets);
}

void attend_parts(int64_t items, int64_t pages, int D, int steps, int64_t taken, int &chunk, int &nchunk) {
    // As many parts as fill the CUs once, beside the `taken` workgroups that run with them: a workgroup's start and end cost as
    // much as several pages.  At most 64 pages, so that long sequences among short ones are spread in any case.
    const int least = waves(D) / steps > 1 ? waves(D) / steps : 1;  // one step a wave
    const int64_t room = PARTS_WG - taken > PARTS_WG / 2 ? PARTS_WG - taken : PARTS_WG / 2;
    const int64_t want = items >= room ? 1 : room / items;
    int64_t c = ((pages + want - 1) / want + least - 1) / least * least;  // the same for every wave
    c = c > 64 ? 64 : c;
    chunk = (int)c;
    nchunk = (int)((pages + c - 1) / c);
}

bool attend_alone(int64_t B, int64_t H, int64_t N, int64_t pages, int D, int dtype, bool prefix) {
    return pages <= ALONE_PAGES && B * H >= ALONE_ITEMS && alone_built(N <= 4 ? 4 : 0, prefix ? prefix_sets(D, B * N, dtype == ST_F32) : 0);
}

}  // namespace fpa
