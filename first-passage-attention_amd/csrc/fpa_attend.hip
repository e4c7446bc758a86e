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
    const int64_t room = CUS - taken > CUS / 2 ? CUS - taken : CUS / 2;
    const int64_t want = items >= room ? 1 : room / items;
    int64_t c = ((pages + want - 1) / want + least - 1) / least * least;  // the same for every wave
    c = c > 64 ? 64 : c;
    chunk = (int)c;
    nchunk = (int)((pages + c - 1) / c);
}

void attend_own(int64_t B, int64_t units, int64_t pages, int D, int steps, int page_bytes, bool prefix, int &least, int &slots, int &nchunk, int64_t &groups) {
    const auto larger = [](int64_t a, int64_t b) { return a > b ? a : b; };
    const auto smaller = [](int64_t a, int64_t b) { return a < b ? a : b; };
    least = waves(D) / steps > 1 ? waves(D) / steps : 1;
    // A part is worth its start, its end and its share of the join from about 16 KB of pages a wave on (B2 H12 D64 L4000: e4m3
    // 14.1 us, fp16 16.2; from 32 KB on 15.8 and 18.7).
    const int worth = waves(D) * (16 << 10) / page_bytes / least * least;
    if (worth > least) least = worth;
    slots = prefix ? CUS / 4 : CUS;
    // What part_pages may come to.  Fewer items than slots: either all parts of all sequences fit the slots, so that one sequence
    // has at most slots / units of them; or, as with more items, a part has LONG_PART pages at least (and `least` in any case).
    const int64_t items = B * units, all = (pages + least - 1) / least, cut = (pages + LONG_PART - 1) / LONG_PART;
    if (!prefix && pages <= 2 * least)
        nchunk = 1;
    else
        nchunk = (int)smaller(all, items < slots ? larger(cut, larger(slots / units, 1)) : cut);
    // Workgroups: in the second case parts of work / LONG_GROUPS pages (or the most that a part may have), rounded up a sequence.
    const int64_t fullest = items * ((pages + most_pages(D) - 1) / most_pages(D));
    groups = smaller(items * cut, larger(LONG_GROUPS, fullest) + items);
    groups = smaller(items < slots ? larger(groups, slots) : groups, items * nchunk);
}

// A wave alone takes its pages one after the other, but needs no fold and no more workgroups than an eighth of the sequences.
// Beside a prefix's parts, which fill the CUs, that is what keeps all in one round (B32 H12 D64 P16381: 42 -> 26 us); by
// themselves short sequences have to be so many that their waves fill the CUs (B33 H12 L742, 400 of them: 33 us alone, 17 in
// workgroups of their own).
bool attend_alone(int64_t B, int64_t H, int64_t N, int64_t pages, int D, int dtype, bool prefix) {
    const bool many = prefix ? pages <= 16 && B * H >= CUS : (pages <= 8 && B * H >= 3 * CUS) || (pages <= 4 && B * H >= 2 * CUS);
    return many && alone_built(N <= 4 ? 4 : 0, prefix ? prefix_sets(D, B * N, dtype == ST_F32) : 0);
}

}  // namespace fpa
