// fpa_attend.h -- First Passage Attention of new tokens against a paged cache.
//
// Query i of N stands at position t = len - N + i of its sequence and attends to the keys s <= t:
//   o_t = sum_s softmax_s(q_t . k_s / sqrt(D) + beta min(0, X_ts - psi_s)) v_s,   X_ts = min_{s < u <= t} phi_u
// (X_tt is +inf).  A shared prefix of PL positions comes before the sequence's own position 0: for its keys
//   X_ts = min(min_{s < u < PL} phi_u, min_{0 <= u <= t} phi_u of the sequence itself),
// so that only the second term differs between the requests, and the rows of all of them form one product
// with the prefix's K and V.
//
// A wave takes its keys in steps of 64, 32 or 16, from the last to the first, and carries the running minimum of phi along;
// what lies between its pages and its queries is one phi_min value a page.  Both cache operands go from HBM straight
// into the registers of the 16x16 MFMA: the pages hold K by rows and V transposed, so that an operand of either
// product is a run of consecutive values.  The next step's K is loaded as soon as this one's scores are formed, the
// next V when this one's is used up.
//
// Two forms of the step:
//   wide  16 rows in the columns of S^T = K Q^T, O^T += V^T P^T (N > 4, and the prefix, there 32 rows where they fit, with every K
//         and V operand used twice).  Of KL = KT / 4 keys a lane group, the key of score register (a, j) of group g is KL g + 4 a + j,
//         so that a lane's weights belong to consecutive keys: as they stand they are the operand of the second product, whose
//         other operand is KL consecutive values of a V^T row.  What belongs to a key (scale, exponents, range minimum) is computed
//         by one lane of each row of 16 and taken from there by DPP.
//   few   up to 4 rows, S = Q K^T with the queries repeated over the 16 rows, so that lane l finds the scores of one key,
//         KT - 1 - l % KT.  Masks, exponentials and scales then cost one operation a step and row where the wide form spends 16
//         on columns that hold no query; the range minimum is a scan over the lanes, and the weights go through
//         LDS into the operand of O = P V.  (B4 H12 D64 L65536 N1 e4m3: 85 us, 135 in the wide form with 4 waves a workgroup.)  One
//         fp32 row runs on the vector unit.
//
// A sequence, and the prefix, is cut into parts of whole pages that run side by side (part_pages, attend_parts), each wave of a
// workgroup taking its share.  Partial results (O, maximum, sum) go to the workspace, and the workgroup that finishes a sequence's
// last part (with a prefix: a tile of its rows') joins them, in the parts' order whoever that is: no second kernel, the same bits
// every time.
//
// What bounds it: HBM on long sequences (B4 H12 D64 L65536 N1 e4m3, 434 MB: 84 us, 5.2 TB/s, as fast as a copy), a chain of start,
// first loads, fold over the waves and join on short ones (B16 H12 D64 L2048 e4m3, 33 MB: 11 us), for many rows behind a prefix in
// e4m3 the vector unit's conversions and exponentials (B64 N4 H8 D128 P8192: 42 us, 8.9 GFLOP).
//
// Softmax statistics and O are fp32.  P is rounded to fp16 for fp16 queries; the running maximum is raised only where a
// weight would pass 2^8, which costs fp16 nothing (what it loses lies 2^-25 below 1) and saves most rescalings; fp32
// queries keep fp32 throughout.  With e4m3 pages the row's power of two of V goes into the logit: the weights
// w_s = p_s 2^e_s are what multiplies the codes, the running maximum is that of w, so that w fills fp16's range whatever
// the scales are, and the sum takes w_s 2^-e_s.
//
// What a query must not see is never multiplied: masked scores are replaced, V rows behind the sequence's end
// are cleared, and an infinity or NaN in a V row that only some of the rows see is left out of the product and
// added for those alone.
#pragma once

#include <type_traits>

#include "fpa_common.h"
#include "fpa_serve.h"

namespace fpa {

namespace {

constexpr int CW = 16;  // query rows of a wave

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// N consecutive cache values of a lane, first as loaded, then as matrix operands.
template <typename TS, int N> struct Raw {
    static constexpr int BYTES = N * (int)sizeof(TS);
    static_assert(BYTES % 4 == 0, "whole words");
    uint32_t w[BYTES / 4];
    // In pieces of 16 bytes (or all of fewer) that lie STRIDE pieces apart.
    template <int STRIDE> __device__ __forceinline__ void load(const TS *p) {
        const char *b = reinterpret_cast<const char *>(p);
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(b + 16 * STRIDE * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
            }
        } else if constexpr (BYTES == 8) {
            const uint2 x = *reinterpret_cast<const uint2 *>(b);
            w[0] = x.x;
            w[1] = x.y;
        } else {
            static_assert(BYTES == 4, "4, 8 or a multiple of 16 bytes");
            w[0] = *reinterpret_cast<const uint32_t *>(b);
        }
    }
    // values 4 i .. 4 i + 3
    __device__ __forceinline__ h4 half4(int i) const {
        if constexpr (sizeof(TS) == 2) {
            const uint2 x = make_uint2(w[2 * i], w[2 * i + 1]);
            return __builtin_bit_cast(h4, x);
        } else {
            static_assert(sizeof(TS) == 1, "fp16 operands come from fp16 or e4m3");
            const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, false);
            const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, true);
            return h4{a[0], a[1], b[0], b[1]};
        }
    }
    __device__ __forceinline__ f32x4 float4_(int i) const {
        if constexpr (sizeof(TS) == 4) {
            return f32x4{__uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1]), __uint_as_float(w[4 * i + 2]),
                         __uint_as_float(w[4 * i + 3])};
        } else {
            static_assert(sizeof(TS) == 1, "fp32 operands come from fp32 or e4m3");
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
            const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
            return f32x4{a[0], a[1], b[0], b[1]};
        }
    }
};

// Matrix operands of N consecutive values per lane: fp16 as h4 quads, fp32 as f32x4 quads.
template <typename TQ> struct Quad;
template <> struct Quad<f16> {
    typedef h4 t;
};
template <> struct Quad<float> {
    typedef f32x4 t;
};
template <typename TQ, typename TS, int N> __device__ __forceinline__ typename Quad<TQ>::t quad(const Raw<TS, N> &r, int i) {
    if constexpr (sizeof(TQ) == 2)
        return r.half4(i);
    else
        return r.float4_(i);
}
// Infinities and NaN are told by the stored bits, as integers: this file is compiled without NaN in mind.
template <typename TS> __device__ __forceinline__ bool beyond_bits(uint32_t bits) {  // of one stored value
    if constexpr (sizeof(TS) == 1) return (bits & 0x7fu) == 0x7fu;
    if constexpr (sizeof(TS) == 2) return (bits & 0x7c00u) == 0x7c00u;
    return (bits & 0x7f800000u) == 0x7f800000u;
}
// Word masks that keep, of N values in pieces of VL whose positions lie 4 VL apart, those at positions below n (from the first's).
template <typename TS, int N, int VL> struct Kept {
    static constexpr int PW = 4 / sizeof(TS), BITS = 8 * sizeof(TS);  // values of a word
    uint32_t w[N / PW];
    __device__ __forceinline__ explicit Kept(int n) {
#pragma unroll
        for (int i = 0; i < N / PW; ++i) {
            const int k = max(n - (i * PW / VL * 4 * VL + i * PW % VL), 0);
            w[i] = k >= PW ? 0xffffffffu : (1u << (k * BITS)) - 1u;
        }
    }
};
// Clears the values that `kept` leaves out and (unless WHOLE) those that are not finite; `some` gets bits where there were
// such among the kept.  An exponent of ones carries into the sign's place when one is added to it.
template <bool WHOLE, typename TS, int N, int VL> __device__ __forceinline__ void clean(Raw<TS, N> &r, const Kept<TS, N, VL> &kept, uint32_t &some) {
    constexpr int PW = Kept<TS, N, VL>::PW;
#pragma unroll
    for (int i = 0; i < N / PW; ++i) {
        r.w[i] &= kept.w[i];
        if constexpr (!WHOLE) {
            uint32_t off;
            if constexpr (sizeof(TS) == 1) {
                off = ((r.w[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                r.w[i] &= ~((off >> 7) * 0xffu);
            } else if constexpr (sizeof(TS) == 2) {
                off = ((r.w[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                r.w[i] &= ~((off >> 15) * 0xffffu);
            } else {
                off = ((r.w[i] & 0x7f800000u) + 0x00800000u) & 0x80000000u;
                r.w[i] &= ~(uint32_t)((int32_t)off >> 31);
            }
            some |= off;
        }
    }
}

constexpr uint32_t BAD = 0xbf800000u;  // -1.0f in place of a row's sum: its table names no page, or its length passes the table
// NaN that the compiler does not see as one (it may drop what it can tell to be NaN).
__device__ __forceinline__ float quiet_nan() {
    uint32_t b = 0x7fc00000u;
    asm("" : "+v"(b));
    return __uint_as_float(b);
}

// The infinity or NaN at vx, or 0 for a finite value.
template <typename TS> __device__ __forceinline__ float not_finite(const TS *vx) {
    if constexpr (sizeof(TS) == 1)
        return beyond_bits<TS>(vx->code) ? quiet_nan() : 0.f;
    else if constexpr (sizeof(TS) == 2)
        return beyond_bits<TS>(*reinterpret_cast<const uint16_t *>(vx)) ? (float)*vx : 0.f;
    else
        return beyond_bits<TS>(*reinterpret_cast<const uint32_t *>(vx)) ? *vx : 0.f;
}

// Features of a lane in the score product: pieces of CH neighbouring ones, 16 bytes of a K row, which the four lane groups take
// in turn, so that one load of the wave reads 64 bytes of a row in a piece (40% fewer L1 accesses at D = 128 in e4m3 than with a
// lane's bytes side by side; the same time, which other things bound).
template <typename TS, int D> constexpr int chunk_of() { return D / 4 < 16 / (int)sizeof(TS) ? D / 4 : 16 / (int)sizeof(TS); }
template <typename TQ, typename TS, int D> __device__ __forceinline__ void load_query(typename Quad<TQ>::t (&q)[D / 16], const TQ *row, int g) {
    constexpr int CH = chunk_of<TS, D>();
#pragma unroll
    for (int i = 0; i < D / 4 / CH; ++i) {
        Raw<TQ, CH> r;
        r.template load<1>(row + CH * (4 * i + g));
#pragma unroll
        for (int k = 0; k < CH / 4; ++k) q[i * (CH / 4) + k] = quad<TQ>(r, k);
    }
}

// acc += A B^T over NQ quads of the contraction (A: row lane % 16, B: column lane % 16, both of the lane
// group's consecutive values).
template <int NQ> __device__ __forceinline__ f32x4 mma(const h4 (&a)[NQ], const h4 (&b)[NQ], f32x4 acc) {
    if constexpr (NQ == 1) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(a[0], b[0], acc, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < NQ; i += 2)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(a[i], a[i + 1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                         __builtin_shufflevector(b[i], b[i + 1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                         acc, 0, 0, 0);
        return acc;
    }
}
template <int NQ> __device__ __forceinline__ f32x4 mma(const f32x4 (&a)[NQ], const f32x4 (&b)[NQ], f32x4 acc) {
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][e], b[i][e], acc, 0, 0, 0);
    return acc;
}

__device__ __forceinline__ float min_groups(float x) {
    x = fminf(x, __shfl_xor(x, 16, 64));
    return fminf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float max_groups(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_groups(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// Length of sequence b, at most what its table holds.
__device__ __forceinline__ int seq_len(const AttendParams &p, int b, bool &bad) {
    const int L = p.lengths[b];
    const int64_t cap = (int64_t)p.P * PG;
    if (L > cap) bad = true;
    return L < 0 ? 0 : (L > cap ? (int)cap : L);
}

// LDS written by the wave's other lanes is read after this (one wave's LDS accesses are in order; the compiler keeps them so).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Inclusive minimum over the lanes 0 .. l.
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_or_inf(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0x7f800000, (int)__float_as_uint(x), CTRL, ROWS, 0xf, false));
}
// KT = 64; 32 or 16: over the lanes of the same half or row.
template <int KT> __device__ __forceinline__ float scan_min(float x) {
    x = fminf(x, dpp_or_inf<0x111, 0xf>(x));  // within rows of 16: 1, 2, 4, 8 lanes down
    x = fminf(x, dpp_or_inf<0x112, 0xf>(x));
    x = fminf(x, dpp_or_inf<0x114, 0xf>(x));
    x = fminf(x, dpp_or_inf<0x118, 0xf>(x));
    if constexpr (KT >= 32) x = fminf(x, dpp_or_inf<0x142, 0xa>(x));  // lane 15 into row 1, 47 into row 3
    if constexpr (KT == 64) x = fminf(x, dpp_or_inf<0x143, 0xc>(x));  // lane 31 into rows 2 and 3
    return x;
}
// The value of the lane below; +inf in the lowest lane.
template <int KT> __device__ __forceinline__ float one_lane_down(float x, int lane) {
    if constexpr (KT == 16) return dpp_or_inf<0x111, 0xf>(x);
    x = dpp_or_inf<0x138, 0xf>(x);
    return KT == 32 && lane == 32 ? pinf() : x;
}
__device__ __forceinline__ float lane_value(float x, int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), l)); }
// The value of lane E of the lane's row of 16 (folded into the instruction that uses it).
template <int E> __device__ __forceinline__ float of_lane(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x150 + E, 0xf, 0xf, true));
}
// Minimum over this lane and those above it in its row of 16.
__device__ __forceinline__ float row_min_above(float x) {
    x = fminf(x, dpp_or_inf<0x101, 0xf>(x));
    x = fminf(x, dpp_or_inf<0x102, 0xf>(x));
    x = fminf(x, dpp_or_inf<0x104, 0xf>(x));
    return fminf(x, dpp_or_inf<0x108, 0xf>(x));
}

// Lanes below 32: x of this lane and of lane + 32; the others: y of lane - 32 and of this lane.  The same for odd and even
// groups of 16.
__device__ __forceinline__ float add_swapped32(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_swapped16(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_self(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(x), (int)__float_as_uint(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_self<0x111, 0xf>(x));
    x = fmaxf(x, dpp_self<0x112, 0xf>(x));
    x = fmaxf(x, dpp_self<0x114, 0xf>(x));
    x = fmaxf(x, dpp_self<0x118, 0xf>(x));
    x = fmaxf(x, dpp_self<0x142, 0xa>(x));
    x = fmaxf(x, dpp_self<0x143, 0xc>(x));
    return lane_value(x, 63);
}
__device__ __forceinline__ float wave_min(float x) { return lane_value(scan_min<64>(x), 63); }

constexpr float SLACK = 8.f;  // a weight may reach 2^SLACK before the running maximum is raised

// Values that another workgroup of this launch reads: agent-scope accesses, which go past the caches that the
// XCDs do not share.
__device__ __forceinline__ void put2(float *p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 get2(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return f32x2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

__device__ __forceinline__ float exp_or_0(float m, float ref) { return fexp2(m - (ref == ninf() ? 0.f : ref)); }

// Workgroups of one round, one a CU; sequences that do not fit one round by parts of fewer than SHORT_PART pages are cut into parts
// of LONG_PART pages at least, for up to ROUNDS of them.
constexpr int CUS = 256, SHORT_PART = 48, LONG_PART = 24, ROUNDS = 4, LONG_GROUPS = ROUNDS * CUS;

// Rows of a prefix tile.
template <int NC> constexpr int tile_rows() { return CW * NC; }

// Waves of a workgroup: as many as two a SIMD (their registers end at 256), so that most sequences need no second part.
constexpr int waves(int D) { return D <= 128 ? 8 : 4; }
// Pages of a part at most: a wave holds the numbers of its own in one register.
constexpr int most_pages(int D) { return 48 * waves(D); }

// Parts of a sequence's own pages: one at least, which may be empty.
__device__ __forceinline__ int own_parts(const AttendParams &p, int L) {
    const int n = ((L + PG - 1) / PG + p.chunk - 1) / p.chunk;
    return n < 1 ? 1 : n;
}

// LDS of a workgroup.
template <int D, int NC> struct Shared {
    static constexpr int NW = waves(D);
    union {
        float fold[NW / 2][NC * CW * D];  // accumulators on their way to another wave
        float alone[NW][4 * D];           // a wave's own rows
    };
    float stat[NW / 2][NC * CW * 2];
    static constexpr int ROWS = tile_rows<NC>();
    float behind[NW];
    uint64_t done[NW];
    int at[NW][2];
    float join[64 * NW][6];
};

// Adds up the parts of rows col0 .. col0 + n - 1 (row col = b N + i) of head h, in order, and writes the output; NT threads.
template <typename TQ, int D, int NT> __device__ void join_rows(const AttendParams &p, int h, int64_t col0, int n, float (*join)[6]) {
    const int tid = thread_x(), H = p.c.H;
    const int64_t R = (int64_t)p.B * H * p.N;
    const int E = n * (D / 4);              // quads of the output
    const int sets = E < NT ? NT / E : 1;   // threads that share a quad's parts
    for (int e0 = 0; e0 < E; e0 += NT) {
        const int e = e0 + tid % min(E, NT), set = E < NT ? tid / E : 0;
        const bool mine = e < E && set < sets;
        const int64_t col = col0 + min(e, E - 1) / (D / 4);
        const int d = e % (D / 4) * 4, b = (int)(col / p.N), i = (int)(col % p.N);
        const int64_t row = ((int64_t)b * H + h) * p.N + i;
        bool bad = false;
        const int own = own_parts(p, seq_len(p, b, bad)), parts = own + p.npchunk;
        float m = ninf(), l = 0.f;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (mine) {
            constexpr int AT_ONCE = 8;  // parts whose loads are in flight together
            for (int k0 = set; k0 < parts; k0 += AT_ONCE * sets) {
                f32x2 s[AT_ONCE], u[AT_ONCE], v[AT_ONCE];
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    const int k = min(k0 + j * sets, parts - 1);
                    const int64_t slot = (int64_t)(k < own ? k : p.nchunk + k - own) * R + row;
                    s[j] = get2(p.ml + 2 * slot);
                    u[j] = get2(p.part + slot * D + d);
                    v[j] = get2(p.part + slot * D + d + 2);
                }
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    if (k0 + j * sets >= parts) break;
                    bad |= __float_as_uint(s[j][1]) == BAD;
                    const float mn = fmaxf(m, s[j][0]), a = exp_or_0(m, mn), w = exp_or_0(s[j][0], mn);
                    l = l * a + s[j][1] * w;
                    x[0] = x[0] * a + u[j][0] * w;
                    x[1] = x[1] * a + u[j][1] * w;
                    x[2] = x[2] * a + v[j][0] * w;
                    x[3] = x[3] * a + v[j][1] * w;
                    m = mn;
                }
            }
        }
        if (sets > 1) {
            __syncthreads();
            join[tid][0] = m;
            join[tid][1] = bad ? __uint_as_float(BAD) : l;
#pragma unroll
            for (int j = 0; j < 4; ++j) join[tid][2 + j] = x[j];
            __syncthreads();
            if (set == 0)
                for (int k = 1; k < sets; ++k) {
                    const float *o = join[k * E + tid];
                    bad |= __float_as_uint(o[1]) == BAD;
                    const float mn = fmaxf(m, o[0]), a = exp_or_0(m, mn), w = exp_or_0(o[0], mn);
                    l = l * a + o[1] * w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = x[j] * a + o[2 + j] * w;
                    m = mn;
                }
        }
        if (mine && set == 0) {
            const bool none = (__float_as_uint(l) << 1) == 0;
            TQ *o = static_cast<TQ *>(p.o) + (int64_t)b * p.so.b + (int64_t)h * p.so.h + (int64_t)i * p.so.t + d;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = (TQ)(bad ? quiet_nan() : none ? 0.f : x[j] / l);
        }
    }
}

// Four neighbouring features of one row's result: the output itself if this part is all of it, else the part's.
template <typename TQ, int D>
__device__ __forceinline__ void put_row(const AttendParams &p, bool whole, int slot, int b, int h, int i, int d, f32x4 x, float m, float l) {
    const bool bad = __float_as_uint(l) == BAD;
    if (whole) {
        const bool none = (__float_as_uint(l) << 1) == 0;
        TQ *o = static_cast<TQ *>(p.o) + (int64_t)b * p.so.b + (int64_t)h * p.so.h + (int64_t)i * p.so.t + d;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (TQ)(bad ? quiet_nan() : none ? 0.f : x[j] / l);
    } else {
        const int64_t at = (int64_t)slot * p.B * p.c.H * p.N + ((int64_t)b * p.c.H + h) * p.N + i;
        put2(p.part + at * D + d, x[0], x[1]);
        put2(p.part + at * D + d + 2, x[2], x[3]);
        if (d == 0) put2(p.ml + 2 * at, m, l);
    }
}

// Counts one part at `count` of `all`: true for the last, which leaves the count at 0 for the next launch.  The part's stores
// are complete: the wave that made them has waited for them.
__device__ __forceinline__ bool last_of(int32_t *count, int all) {
    const int before = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before + 1 < all) return false;
    __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}
// With a prefix the rows are joined by its tiles: the prefix's parts, and those of every sequence with a row in the tile.
template <int ROWS> __device__ __forceinline__ bool last_of_tile(const AttendParams &p, int h, int tile) {
    const int64_t c0 = (int64_t)tile * ROWS, c1 = min(c0 + ROWS, (int64_t)p.B * p.N) - 1;
    const int b0 = (int)(c0 / p.N), b1 = (int)(c1 / p.N), nrt = (p.N + CW - 1) / CW;
    int own = b1 - b0 + 1;
    if (p.nchunk > 1) {
        own = 0;
        bool lost = false;
#pragma unroll 4
        for (int b = b0; b <= b1; ++b) own += own_parts(p, seq_len(p, b, lost));
    }
    const int tiles = (int)(((int64_t)p.B * p.N + ROWS - 1) / ROWS);
    return last_of(p.counts + (int64_t)h * tiles + tile, p.npchunk + own * nrt);
}
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int N, typename F> __device__ __forceinline__ void unrolled(F &&f) {
    if constexpr (N > 0) {
        unrolled<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

// A wave's share of a part, in steps of KT keys (HT a page): steps [T0, T1) of the segment.
template <int NW, int HT, bool ALONE> __device__ __forceinline__ void wave_steps(int ps, int pe, int wave, int &T0, int &T1) {
    const int n = pe > ps ? (pe - ps) * HT : 0, per = ALONE ? n : (n + NW - 1) / NW;
    T0 = ps * HT + (ALONE ? 0 : min(wave * per, n));
    if constexpr (ALONE) asm("" : "+s"(T0));  // a constant 0 here makes the compiler rearrange the step loops, with hundreds of spills
    T1 = min(T0 + per, ps * HT + n);
}

// The page numbers of a wave's pages [ws, we) (at most 64), one a lane; pages that do not exist become 0 and are told.
__device__ __forceinline__ int page_numbers(const AttendParams &p, const int32_t *table, int ws, int we, int lane, bool &missing) {
    int page = 0;
    if (ws + lane < we) {
        page = table[ws + lane];
        if ((uint32_t)page >= (uint64_t)p.c.n) {
            missing = true;
            page = 0;
        }
    }
    return page;
}
// min of phi_min over the pages k0, k0 + step, .. < k1 of this lane.
__device__ __forceinline__ float lane_min(const AttendParams &p, const int32_t *table, int h, int k0, int k1, int step, bool &missing) {
    float m = pinf();
#pragma unroll 4
    for (int k = k0; k < k1; k += step) {
        const int page = table[k];
        const bool there = (uint32_t)page < (uint64_t)p.c.n;
        missing |= !there;
        const float x = p.c.phi_min[(int64_t)(there ? page : 0) * p.c.H + h];
        m = there ? fminf(m, x) : m;
    }
    return m;
}

// After a workgroup's own parts: `writer` waves have stored one of sequence b, head h, and join what is complete with it.  Every
// thread of the workgroup comes here.
template <typename TQ, int D, typename SH> __device__ void own_done(const AttendParams &p, bool writer, int b, int h, SH &sh) {
    constexpr int NW = waves(D), ROWS = SH::ROWS;
    const int lane = thread_x() % 64, wave = uni(thread_x() / 64);
    if (writer) stores_done();
    if (p.npchunk == 0) {
        bool lost = false;
        if (writer && lane == 0)
            sh.done[0] = last_of(p.counts + (int64_t)b * p.c.H + h, own_parts(p, seq_len(p, b, lost)) * ((p.N + CW - 1) / CW));
        __syncthreads();
        if (sh.done[0]) join_rows<TQ, D, 64 * NW>(p, h, (int64_t)b * p.N, p.N, sh.join);
        return;
    }
    // the tiles that hold rows of the sequence, 64 at a time
    const int t0 = (int)((int64_t)b * p.N / ROWS), t1 = (int)(((int64_t)b * p.N + p.N - 1) / ROWS);
    const int most = (p.N + ROWS - 1) / ROWS + 1;
    for (int k0 = 0; k0 < most; k0 += 64) {
        const int t = t0 + k0 + lane;
        const uint64_t last = __ballot(writer && t <= t1 && last_of_tile<ROWS>(p, h, min(t, t1)));
        if (lane == 0) {
            sh.done[wave] = last;
            sh.at[wave][0] = h;
            sh.at[wave][1] = t0 + k0;
        }
        __syncthreads();
        for (int w = 0; w < NW; ++w)
            for (uint64_t left = sh.done[w]; left; left &= left - 1) {
                const int64_t c0 = (int64_t)(sh.at[w][1] + __builtin_ctzll(left)) * ROWS;
                join_rows<TQ, D, 64 * NW>(p, sh.at[w][0], c0, (int)min((int64_t)ROWS, (int64_t)p.B * p.N - c0), sh.join);
            }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// few
// ---------------------------------------------------------------------------
// Keys of a step: 64 rows of K and of V where that leaves room for the next step's (KT * D * sizeof(TS) / 256 registers
// each), for their conversions and the other rows, else 32 or 16; the upper lanes then repeat the lower ones.
template <typename TQ, typename TS, int D, int NR> constexpr int few_keys() {
    const int w = D * (sizeof(TS) > sizeof(TQ) / 2 ? (int)sizeof(TS) : (int)sizeof(TQ) / 2) * (NR > 1 ? 2 : 1);
    return w <= 256 && D <= 128 ? 64 : w <= 512 ? 32 : 16;
}

// ALONE: the wave takes the whole part by itself (and the other waves of the workgroup other sequences).
template <typename TQ, typename TS, int D, int NR, bool ALONE, typename SH>
__device__ __forceinline__ void few_rows(const AttendParams &p, int b, int h, int part, SH &sh, TQ (*weights)[NR * PG]) {
    typedef typename Quad<TQ>::t quad_t;
    constexpr int DG = D / 4, ND = D / 16, NW = waves(D);
    constexpr int KT = few_keys<TQ, TS, D, NR>(), KL = KT / 4, A = KT / 16, HT = PG / KT;
    constexpr int CH = chunk_of<TS, D>(), VL = KL < 16 / (int)sizeof(TS) ? KL : 16 / (int)sizeof(TS);  // values of a piece of K and V
    // Value e of a V run is key 4 VL (e / VL) + VL g + e % VL of the step.
    // One fp32 row: the fp32 MFMA would take 15 idle rows along, 8 times the cycles that the same operands take on the vector
    // unit, each lane summing over its own features or keys.
    constexpr bool ONE = sizeof(TQ) == 4 && NR == 1;
    const int tid = thread_x(), lane = tid % 64, wave = uni(tid / 64), c = lane % 16, g = lane / 16;
    const int H = p.c.H;
    bool missing = false;
    const int L = uni(seq_len(p, b, missing));
    const int npg = (L + PG - 1) / PG;
    const int ps = part * p.chunk, pe = min(ps + p.chunk, npg);
    const int32_t *table = p.table + (int64_t)b * p.stable;
    const int t0 = L - p.N;                      // position of row 0
    const int sees_all = t0 >= 0 ? t0 + 1 : 0;   // positions that every row sees
    const int pf = sees_all / PG;
    int T0, T1;
    wave_steps<NW, HT, ALONE>(ps, pe, wave, T0, T1);
    const int ws = T0 / HT, we = (T1 + HT - 1) / HT;  // the pages they are on
    const int cut = T1 % HT * KT;                     // keys of the last that are the wave's, 0: all
    // Everything that names a page first, then what those name: two trips to memory before the first scores.
    const int pages = page_numbers(p, table, ws, T0 < T1 ? we : ws, lane, missing);
    const bool far = pf > (ALONE ? we : ps) + PG;  // more whole pages behind than one load of the wave covers
    const int near_end = min(far && !ALONE ? min(pe, pf) : pf, we + PG);
    const int behind_page = page_numbers(p, table, we, T0 < T1 ? near_end : 0, lane, missing);
    const int part_page = page_numbers(p, table, max(we, pf), T0 < T1 ? npg : 0, lane, missing);  // at most two
    float mine = T0 < T1 && we + lane < near_end ? p.c.phi_min[(int64_t)behind_page * H + h] : pinf();
    auto head_page = [&](int pg) { return (int64_t)__builtin_amdgcn_readlane(pages, pg - ws) * H + h; };
    auto place = [&](int T) { return head_page(T / HT) * PG + T % HT * KT; };  // step T's first position in the pool, for this head

    const int key = KT - 1 - lane % KT;
    Raw<TS, DG> kr[A];
    Raw<TS, KL> vr[ND];
    float phv = 0.f, psv = 0.f;
    int ke = 0, ve = 0;
    auto load_k = [&](int64_t at) __attribute__((always_inline)) {
        const TS *kp = static_cast<const TS *>(p.c.k) + at * D;
#pragma unroll
        for (int a = 0; a < A; ++a) kr[a].template load<4>(kp + (KT - 1 - 16 * a - c) * D + g * CH);
        phv = p.c.phi[at + key];
        psv = p.c.psi[at + key];
        if constexpr (sizeof(TS) == 1) ke = p.c.k_exp[at + key];
    };
    auto load_v = [&](int64_t at) __attribute__((always_inline)) {
        const TS *vp = static_cast<const TS *>(p.c.v) + at / PG * (PG * D) + at % PG;
        if constexpr (sizeof(TS) == 1) ve = p.c.v_exp[at + key];
#pragma unroll
        for (int d = 0; d < ND; ++d) vr[d].template load<4>(vp + (16 * d + c) * PG + VL * g);
    };
    const int first = min(T1, (L + KT - 1) / KT) - 1;  // steps behind the last position hold nothing
    if (T0 <= first) {
        const int64_t at = place(first);
        load_k(at);
        load_v(at);
    }

    quad_t qv[DG / 4];
    {
        const int i = NR == 1 ? 0 : c % NR;
        load_query<TQ, TS, D>(qv, static_cast<const TQ *>(p.q) + (int64_t)b * p.sq.b + (int64_t)h * p.sq.h + (int64_t)min(i, p.N - 1) * p.sq.t, g);
    }  // rows past N repeat the last: never written
    const float beta2 = p.beta[h] * LOG2E;

    // min of phi from the wave's pages on: whole pages, those behind the part by all waves together where there are many, then the at most
    // two pages that some rows see in part
    float carry[NR];
    {
        if (far && T0 < T1) mine = fminf(mine, lane_min(p, table, h, we + PG + lane, ALONE ? pf : min(pe, pf), 64, missing));
        mine = wave_min(mine);
        if (!ALONE && far) {
            const float m = wave_min(lane_min(p, table, h, pe + tid, pf, 64 * NW, missing));
            if (lane == 0) sh.behind[wave] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) mine = fminf(mine, sh.behind[w]);
        }
#pragma unroll
        for (int j = 0; j < NR; ++j) carry[j] = mine;
        if (T0 < T1) {
            if (HT > 1 && cut) {  // the rest of a page that the wave shares
                const int64_t ph = head_page(we - 1);
                const float f = p.c.phi[ph * PG + lane];
                const int pos = (we - 1) * PG + lane;
#pragma unroll
                for (int j = 0; j < NR; ++j) carry[j] = fminf(carry[j], wave_min(lane >= cut && pos <= min(t0 + j, L - 1) ? f : pinf()));
            }
            for (int k = max(we, pf); k < npg; ++k) {
                const int64_t ph = (int64_t)__builtin_amdgcn_readlane(part_page, k - max(we, pf)) * H + h;
                const float f = p.c.phi[ph * PG + lane];
#pragma unroll
                for (int j = 0; j < NR; ++j) carry[j] = fminf(carry[j], wave_min(k * PG + lane <= min(t0 + j, L - 1) ? f : pinf()));
            }
        }
    }

    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m[NR], l[NR];  // the maximum is the wave's, the sum the lane's
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        m[j] = ninf();
        l[j] = 0.f;
    }
    TQ *wl = weights[wave];

    auto step = [&](auto tail_tag, auto more_tag, int T) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail_tag)::value, MORE = decltype(more_tag)::value;  // MORE: another step follows
        const int pos = T * KT + key;
        const int64_t next = MORE ? place(T - 1) : 0;
        f32x4 s[A];
#pragma unroll
        for (int a = 0; a < A; ++a) {
            quad_t kq[DG / 4];
#pragma unroll
            for (int k = 0; k < DG / 4; ++k) kq[k] = quad<TQ>(kr[a], k);
            if constexpr (ONE) {
                s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < DG / 4; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[a][e] += kq[k][e] * qv[k][e];
                s[a][0] = (s[a][0] + s[a][1]) + (s[a][2] + s[a][3]);
                __builtin_amdgcn_sched_barrier(0);  // one tile's conversions at a time: all at once do not fit the registers
            } else {
                s[a] = mma<DG / 4>(qv, kq, f32x4{0.f, 0.f, 0.f, 0.f});
            }
        }
        if constexpr (ONE) {  // over the lane groups: group g ends with the sums of tile g mod A
            if constexpr (A == 4) {
                s[0][0] = add_swapped32(s[0][0], s[2][0]);
                s[1][0] = add_swapped32(s[1][0], s[3][0]);
                s[0][0] = add_swapped16(s[0][0], s[1][0]);
            } else {
                s[0][0] = add_swapped32(s[0][0], s[0][0]);
                if constexpr (A == 2) s[1][0] = add_swapped32(s[1][0], s[1][0]);
                s[0][0] = add_swapped16(s[0][0], s[A == 2 ? 1 : 0][0]);
            }
        }
        float t[NR];
        if constexpr (!TAIL) {
            const float inc = scan_min<KT>(phv), x = one_lane_down<KT>(inc, lane), all = lane_value(inc, KT - 1);
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                t[j] = fminf(x, carry[j]);
                carry[j] = fminf(carry[j], all);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                const float inc = scan_min<KT>(pos <= min(t0 + j, L - 1) ? phv : pinf());
                t[j] = fminf(one_lane_down<KT>(inc, lane), carry[j]);
                carry[j] = fminf(carry[j], lane_value(inc, KT - 1));
            }
        }
        const float sc = sizeof(TS) == 1 ? p.sc2 * pow2(ke) : p.sc2;
        bool up = false;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            float sj = s[0][j];  // lane group g has the keys of tile g mod A
            if constexpr (A == 2 && !ONE) sj = g % 2 ? s[1][j] : sj;
            if constexpr (A == 4 && !ONE) sj = g < 2 ? (g == 0 ? sj : s[1][j]) : (g == 2 ? s[2][j] : s[3][j]);
            t[j] = (sizeof(TS) == 1 ? sj * sc + (float)ve : sj * sc) + beta2 * fminf(t[j] - psv, 0.f);
            if (TAIL && pos > min(t0 + j, L - 1)) t[j] = ninf();
            up |= t[j] > m[j] + SLACK;
        }
        if constexpr (MORE) load_k(next);
        if (__any(up)) {  // rare after the first steps
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                const float mn = fmaxf(m[j], wave_max(t[j]));
                const float alpha = exp_or_0(m[j], mn);
                m[j] = mn;
                l[j] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) acc[d][j] *= alpha;
            }
        }
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const float w = exp_or_0(t[j], m[j]);
            wl[j * PG + key] = (TQ)w;
            t[j] = w;
            l[j] += sizeof(TS) == 1 ? w * pow2(-ve) : w;
        }
        wave_sync();
        quad_t pq[A];
#pragma unroll
        for (int a = 0; a < A; ++a) pq[a] = *reinterpret_cast<const quad_t *>(wl + (NR == 1 ? 0 : c % NR) * PG + 4 * VL * (4 * a / VL) + VL * g + 4 * a % VL);
        wave_sync();
        uint32_t some = 0;
        const Kept<TS, KL, VL> kept(TAIL ? L - T * KT - VL * g : KT);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if constexpr (TAIL) clean<NR == 1>(vr[d], kept, some);
            quad_t vq[A];
#pragma unroll
            for (int a = 0; a < A; ++a) vq[a] = quad<TQ>(vr[d], a);
            if constexpr (ONE) {
#pragma unroll
                for (int a = 0; a < A; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][0] += vq[a][e] * pq[a][e];
                __builtin_amdgcn_sched_barrier(0);
            } else {
                acc[d] = mma<A>(pq, vq, acc[d]);
            }
        }
        if (TAIL && NR > 1 && __any(some != 0)) {  // infinities and NaN, for the rows that see them
            const int64_t at = place(T);
            const TS *vp = static_cast<const TS *>(p.c.v) + at / PG * (PG * D) + at % PG;
            for (int e = 0; e < KT; ++e) {
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const float y = not_finite(vp + (16 * d + c) * PG + e);
#pragma unroll
                    for (int j = 0; j < NR; ++j) {
                        const float w = __shfl(t[j], KT - 1 - e, 64);
                        if (T * KT + e <= t0 + j && __float_as_uint(y) != 0) acc[d][j] += w * y;
                    }
                }
            }
        }
        if constexpr (MORE) load_v(next);
    };
    const std::true_type yes{};
    const std::false_type no{};
    int T = first;
    for (; T > T0 && (T + 1) * KT > sees_all; --T) step(yes, yes, T);
    for (; T > T0; --T) step(no, yes, T);
    if (T == T0) {
        if ((T + 1) * KT > sees_all)
            step(yes, no, T);
        else
            step(no, no, T);
    }

    const bool bad = __any(missing);
    if constexpr (ONE) {
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d][0] = sum_groups(acc[d][0]);
    }
#pragma unroll
    for (int j = 0; j < NR; ++j) {
#pragma unroll
        for (int o = 1; o < KT; o <<= 1) l[j] += __shfl_xor(l[j], o, 64);
        if (bad) l[j] = __uint_as_float(BAD);
    }
    // The waves' results together, the upper half into the lower, down to wave 0.
#pragma unroll
    for (int from = ALONE ? 0 : NW / 2; from >= 1; from /= 2) {
        __syncthreads();
        if (wave >= from && wave < 2 * from) {
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                if (lane == 0) {
                    sh.stat[wave - from][2 * j] = m[j];
                    sh.stat[wave - from][2 * j + 1] = l[j];
                }
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    if (g == d % 4) sh.fold[wave - from][j * D + 16 * d + c] = acc[d][j];
            }
        }
        __syncthreads();
        if (wave < from) {
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                const float m2 = sh.stat[wave][2 * j], l2 = sh.stat[wave][2 * j + 1], mn = fmaxf(m[j], m2);
                const float a = exp_or_0(m[j], mn), w = exp_or_0(m2, mn);
                const bool lost = __float_as_uint(l[j]) == BAD || __float_as_uint(l2) == BAD;
                m[j] = mn;
                l[j] = lost ? __uint_as_float(BAD) : l[j] * a + l2 * w;
#pragma unroll
                for (int d = 0; d < ND; ++d) acc[d][j] = acc[d][j] * a + sh.fold[wave][j * D + 16 * d + c] * w;
            }
        }
    }
    const bool whole = p.npchunk == 0 && (ALONE || own_parts(p, L) == 1);
    if (ALONE || wave == 0) {
        float *row = ALONE ? sh.alone[wave] : sh.fold[1];
#pragma unroll
        for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (g == d % 4) row[j * D + 16 * d + c] = acc[d][j];
        wave_sync();
#pragma unroll
        for (int j = 0; j < NR; ++j)
            if (j < p.N && 4 * lane < D)
                put_row<TQ, D>(p, whole, part, b, h, j, 4 * lane, *reinterpret_cast<const f32x4 *>(&row[j * D + 4 * lane]), m[j], l[j]);
    }
    if (!whole) own_done<TQ, D>(p, ALONE || wave == 0, b, h, sh);
}

// ---------------------------------------------------------------------------
// wide
// ---------------------------------------------------------------------------
template <typename TQ, typename TS, int D, int NC> constexpr int wide_keys() {
    return D * (int)sizeof(TS) <= 128 && D * (int)sizeof(TQ) <= 256 && NC == 1 ? 64 : D * (int)sizeof(TS) * NC <= 256 ? 32 : 16;
}

template <typename TQ, typename TS, int D, int NC, bool PRE, bool ALONE, typename SH>
__device__ __forceinline__ void wide_rows(const AttendParams &p, int b0, int h, int tile, int part, SH &sh) {
    typedef typename Quad<TQ>::t quad_t;
    constexpr int DG = D / 4, ND = D / 16, ROWS = tile_rows<NC>(), NW = waves(D);
    // Keys of a step: as many of a page as leave room for the operands of the next step (KT * D * sizeof(TS) / 256 registers
    // each for K and V), the accumulators and the queries.
    constexpr int KT = wide_keys<TQ, TS, D, NC>(), KL = KT / 4, A = KT / 16, HT = PG / KT;  // KL of a lane, HT steps a page
    constexpr int CH = chunk_of<TS, D>();
    static_assert(PRE || NC == 1, "a sequence's own rows in tiles of 16");
    const int tid = thread_x(), lane = tid % 64, wave = uni(tid / 64), c = lane % 16, g = lane / 16;
    const int H = p.c.H;
    bool missing = false;                 // a page of the segment that its table does not name: every row's
    bool bad[NC];                         // of the lane's row
    bool valid[NC];
    int sb[NC], si[NC], last[NC];         // sequence, query, last position of the segment that the row sees (-1: none)
    int npg, pf, lmax, sees_all;          // pages of the segment, pages that every row sees whole, the largest `last`; positions all rows see
    const int32_t *table;
    const int64_t rows = PRE ? (int64_t)p.B * p.N : p.N;
    if constexpr (PRE) {
        table = p.prefix;
        npg = (p.PL + PG - 1) / PG;
        sees_all = p.PL;
        lmax = p.PL - 1;
    } else {
        table = p.table + (int64_t)b0 * p.stable;
        const int L = uni(seq_len(p, b0, missing)), tmin = L - p.N + tile * ROWS;
        lmax = min(tmin + ROWS, L) - 1;
        npg = lmax >= 0 ? lmax / PG + 1 : 0;
        sees_all = tmin >= 0 ? tmin + 1 : 0;
    }
    pf = sees_all / PG;
    const int chunk = PRE ? p.pchunk : p.chunk;
    const int ps = part * chunk, pe = min(ps + chunk, npg);
    int T0, T1;
    wave_steps<NW, HT, ALONE>(ps, pe, wave, T0, T1);
    const int ws = T0 / HT, we = (T1 + HT - 1) / HT;  // the pages they are on
    const int cut = T1 % HT * KT;                     // keys of the last that are the wave's, 0: all
    const int pages = page_numbers(p, table, ws, T0 < T1 ? we : ws, lane, missing);
    const bool far = pf > (ALONE ? we : ps) + PG;
    const int near_end = min(far && !ALONE ? min(pe, pf) : pf, we + PG);
    const int behind_page = page_numbers(p, table, we, T0 < T1 ? near_end : 0, lane, missing);
    const int part_page = page_numbers(p, table, max(we, pf), T0 < T1 ? npg : 0, lane, missing);
    float mine = T0 < T1 && we + lane < near_end ? p.c.phi_min[(int64_t)behind_page * H + h] : pinf();
    auto head_page = [&](int pg) { return (int64_t)__builtin_amdgcn_readlane(pages, pg - ws) * H + h; };

    // step T: keys KT T .. KT T + KT - 1 of the segment
    Raw<TS, DG> kr[A];
    Raw<TS, KL> vr[ND];
    // phi, psi and the exponents of one key a lane: of group g's keys, that of number c mod KL
    float phv = 0.f, psv = 0.f;
    int ke = 0, ve = 0;
    auto place = [&](int T) { return head_page(T / HT) * PG + T % HT * KT; };  // the step's first position in the pool, for this head
    auto load_k = [&](int64_t at) __attribute__((always_inline)) {
        const TS *kp = static_cast<const TS *>(p.c.k) + at * D;
#pragma unroll
        for (int a = 0; a < A; ++a) kr[a].template load<4>(kp + (KL * (c / 4) + 4 * a + c % 4) * D + g * CH);
    };
    auto load_s = [&](int64_t at) __attribute__((always_inline)) {
        const int64_t i = at + KL * g + c % KL;
        phv = p.c.phi[i];
        psv = p.c.psi[i];
        if constexpr (sizeof(TS) == 1) {
            ke = p.c.k_exp[i];
            ve = p.c.v_exp[i];
        }
    };
    auto load_v = [&](int64_t at) __attribute__((always_inline)) {
        const TS *vp = static_cast<const TS *>(p.c.v) + at / PG * (PG * D) + at % PG;
#pragma unroll
        for (int d = 0; d < ND; ++d) vr[d].template load<1>(vp + (16 * d + c) * PG + KL * g);
    };
    const int first = min(T1, lmax >= 0 ? lmax / KT + 1 : 0) - 1;  // steps behind the last position hold nothing
    if (T0 <= first) {
        const int64_t at = place(first);
        load_k(at);
        load_s(at);
        load_v(at);
    }

    quad_t qv[NC][DG / 4];
    float carry[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int64_t col = (int64_t)tile * ROWS + k * CW + c;
        valid[k] = col < rows;
        sb[k] = PRE ? (valid[k] ? (int)(col / p.N) : 0) : b0;
        si[k] = valid[k] ? (int)(PRE ? col % p.N : col) : 0;
        bad[k] = false;
        const int t = seq_len(p, sb[k], bad[k]) - p.N + si[k];
        last[k] = valid[k] && t >= 0 ? (PRE ? lmax : t) : -1;
        // columns past the rows repeat one: never written
        load_query<TQ, TS, D>(qv[k], static_cast<const TQ *>(p.q) + (int64_t)sb[k] * p.sq.b + (int64_t)h * p.sq.h + (int64_t)si[k] * p.sq.t, g);
        carry[k] = pinf();
        if constexpr (PRE) {  // min of the sequence's own phi up to t, the lane groups taking the whole pages in turn
            const int32_t *tb = p.table + (int64_t)sb[k] * p.stable;
            const int full = t >= 0 ? (t + 1) / PG : 0, rest = t >= 0 ? (t + 1) % PG : 0;
            carry[k] = lane_min(p, tb, h, g, full, 4, bad[k]);
            if (rest > 0) {
                const int page = tb[full];
                const bool there = (uint32_t)page < (uint64_t)p.c.n;
                bad[k] |= !there;
                const float *ph = p.c.phi + ((int64_t)(there ? page : 0) * H + h) * PG + 16 * g;
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f32x4 f = *reinterpret_cast<const f32x4 *>(ph + e);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (16 * g + e + j < rest) carry[k] = fminf(carry[k], f[j]);
                }
            }
        }
    }
    const float beta2 = p.beta[h] * LOG2E;
    {
        if (far && T0 < T1) mine = fminf(mine, lane_min(p, table, h, we + PG + lane, ALONE ? pf : min(pe, pf), 64, missing));
        mine = wave_min(mine);
        if (!ALONE && far) {
            const float mb = wave_min(lane_min(p, table, h, pe + tid, pf, 64 * NW, missing));
            if (lane == 0) sh.behind[wave] = mb;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; ++i) mine = fminf(mine, sh.behind[i]);
        }
        if (T0 < T1) {
            // the rest of a page that the wave shares, then at most two pages that some rows see in part
            for (int k = HT > 1 && cut ? -1 : max(we, pf); k < npg; k = k < 0 ? max(we, pf) : k + 1) {
                const int64_t page = k < 0 ? head_page(we - 1) : (int64_t)__builtin_amdgcn_readlane(part_page, k - max(we, pf)) * H + h;
                const int pos = (k < 0 ? we - 1 : k) * PG + 16 * g, from = k < 0 ? (we - 1) * PG + cut : 0;
                const float *ph = p.c.phi + page * PG + 16 * g;
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const f32x4 f = *reinterpret_cast<const f32x4 *>(ph + e);
#pragma unroll
                    for (int q = 0; q < NC; ++q)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (pos + e + j >= from && pos + e + j <= last[q]) carry[q] = fminf(carry[q], f[j]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NC; ++k) carry[k] = fminf(min_groups(carry[k]), mine);
    }

    f32x4 acc[NC][ND];
    float m[NC], l[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        m[k] = ninf();
        l[k] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[k][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    auto step = [&](auto tail_tag, auto more_tag, int T) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail_tag)::value, MORE = decltype(more_tag)::value;  // MORE: another step follows
        const int key0 = T * KT + KL * g;  // the lane's first key
        const int64_t next = MORE ? place(T - 1) : 0;
        f32x4 s[NC][A];
#pragma unroll
        for (int a = 0; a < A; ++a) {
            quad_t kq[DG / 4];
#pragma unroll
            for (int i = 0; i < DG / 4; ++i) kq[i] = quad<TQ>(kr[a], i);
#pragma unroll
            for (int k = 0; k < NC; ++k) s[k][a] = mma<DG / 4>(kq, qv[k], f32x4{0.f, 0.f, 0.f, 0.f});
        }
        if constexpr (MORE) load_k(next);
        // Per key, in the lane that holds it: scale, exponents; the range minimum over the group's later keys.  A score takes its
        // key's from there.
        const float sc = sizeof(TS) == 1 ? p.sc2 * pow2(ke) : p.sc2, vz = (float)ve, vinv = sizeof(TS) == 1 ? pow2(-ve) : 1.f, psi = psv;
        float inner = 0.f, behind = 0.f, all = 0.f;  // the same for every row outside the tail
        if constexpr (!TAIL) {
            const float inc = row_min_above(KL == 16 || c < KL ? phv : pinf());
            inner = fminf(dpp_or_inf<0x101, 0xf>(inc) - psv, 0.f);
            const float r3 = lane_value(inc, 48), r2 = fminf(lane_value(inc, 32), r3), r1 = fminf(lane_value(inc, 16), r2);
            behind = g == 3 ? pinf() : g == 2 ? r3 : g == 1 ? r2 : r1;
            all = fminf(lane_value(inc, 0), r1);
        }
        float t[NC][KL];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float x[KL];
            if constexpr (TAIL) {  // every row its own keys
                float r = pinf();
                unrolled<KL>([&](auto i) __attribute__((always_inline)) {
                    constexpr int e = KL - 1 - decltype(i)::value;
                    x[e] = fminf(r - of_lane<e>(psi), 0.f);
                    const float f = of_lane<e>(phv);
                    r = fminf(r, key0 + e <= last[k] ? f : pinf());
                });
                const float r1 = __shfl_down(r, 16, 64), r2 = __shfl_down(r, 32, 64), r3 = __shfl_down(r, 48, 64);
                behind = pinf();
                if (g < 3) behind = r1;
                if (g < 2) behind = fminf(behind, r2);
                if (g < 1) behind = fminf(behind, r3);
                all = __shfl(fminf(behind, r), c, 64);
            }
            const float low = fminf(behind, carry[k]);
            carry[k] = fminf(carry[k], all);
            unrolled<KL>([&](auto i) __attribute__((always_inline)) {
                constexpr int e = decltype(i)::value;
                float z = sizeof(TS) == 1 ? s[k][e / 4][e % 4] * of_lane<e>(sc) + of_lane<e>(vz) : s[k][e / 4][e % 4] * sc;
                float u = low - of_lane<e>(psi);
                if constexpr (TAIL)
                    u = fminf(u, x[e]);
                else
                    u = fminf(u, of_lane<e>(inner));
                t[k][e] = z + beta2 * u;
                if (TAIL && key0 + e > last[k]) t[k][e] = ninf();
            });
        }
        if constexpr (MORE) load_s(next);
        quad_t pq[NC][A];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float mt = t[k][0];
#pragma unroll
            for (int e = 1; e < KL; ++e) mt = fmaxf(mt, t[k][e]);
            if (__any(mt > m[k] + SLACK)) {  // rare after the first steps
                const float mn = fmaxf(m[k], max_groups(mt)), alpha = exp_or_0(m[k], mn);
                m[k] = mn;
                l[k] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[k][d][j] *= alpha;
            }
            const float ref = m[k] == ninf() ? 0.f : m[k];
            unrolled<KL>([&](auto i) __attribute__((always_inline)) {
                constexpr int e = decltype(i)::value;
                t[k][e] = fexp2(t[k][e] - ref);
                l[k] += sizeof(TS) == 1 ? t[k][e] * of_lane<e>(vinv) : t[k][e];
                pq[k][e / 4][e % 4] = (TQ)t[k][e];
            });
        }
        uint32_t some = 0;
        const Kept<TS, KL, KL> kept(TAIL ? lmax + 1 - key0 : KT);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if constexpr (TAIL) clean<PRE>(vr[d], kept, some);
            quad_t vq[A];
#pragma unroll
            for (int a = 0; a < A; ++a) vq[a] = quad<TQ>(vr[d], a);
#pragma unroll
            for (int k = 0; k < NC; ++k) acc[k][d] = mma<A>(vq, pq[k], acc[k][d]);
        }
        if (TAIL && !PRE && __any(some != 0)) {  // infinities and NaN, for the rows that see them
            const int64_t at = place(T);
            const TS *vp = static_cast<const TS *>(p.c.v) + at / PG * (PG * D) + at % PG;
            for (int e = 0; e < KT; ++e) {
                float w = t[0][0];
#pragma unroll
                for (int k = 1; k < KL; ++k) w = e % KL == k ? t[0][k] : w;
                w = __shfl(w, e / KL * 16 + c, 64);
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float y = not_finite(vp + (16 * d + 4 * g + j) * PG + e);
                        if (T * KT + e <= last[0] && __float_as_uint(y) != 0) acc[0][d][j] += w * y;
                    }
            }
        }
        if constexpr (MORE) load_v(next);
    };
    const std::true_type yes{};
    const std::false_type no{};
    int T = first;
    for (; T > T0 && (T + 1) * KT > sees_all; --T) step(yes, yes, T);
    for (; T > T0; --T) step(no, yes, T);
    if (T == T0) {
        if ((T + 1) * KT > sees_all)
            step(yes, no, T);
        else
            step(no, no, T);
    }

    const bool lost = __any(missing);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        l[k] = sum_groups(l[k]);
        if (last[k] < 0) {  // a row that sees nothing: whole pages are not masked for it
            m[k] = ninf();
            l[k] = 0.f;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[k][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (lost || max_groups(bad[k] ? 1.f : 0.f) > 0.f) l[k] = __uint_as_float(BAD);
    }
    // The waves' results together, the upper half into the lower, down to wave 0 (lane by lane: every wave has the same rows).
#pragma unroll
    for (int from = ALONE ? 0 : NW / 2; from >= 1; from /= 2) {
        __syncthreads();
        if (wave >= from && wave < 2 * from) {
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                if (g == 0) {
                    sh.stat[wave - from][2 * (k * CW + c)] = m[k];
                    sh.stat[wave - from][2 * (k * CW + c) + 1] = l[k];
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&sh.fold[wave - from][((k * ND + d) * 64 + lane) * 4]) = acc[k][d];
            }
        }
        __syncthreads();
        if (wave < from) {
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const float m2 = sh.stat[wave][2 * (k * CW + c)], l2 = sh.stat[wave][2 * (k * CW + c) + 1], mn = fmaxf(m[k], m2);
                const float a = exp_or_0(m[k], mn), w = exp_or_0(m2, mn);
                const bool b2 = __float_as_uint(l[k]) == BAD || __float_as_uint(l2) == BAD;
                m[k] = mn;
                l[k] = b2 ? __uint_as_float(BAD) : l[k] * a + l2 * w;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const f32x4 o = *reinterpret_cast<const f32x4 *>(&sh.fold[wave][((k * ND + d) * 64 + lane) * 4]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[k][d][j] = acc[k][d][j] * a + o[j] * w;
                }
            }
        }
    }
    bool over = false;
    const bool whole = !PRE && p.npchunk == 0 && (ALONE || own_parts(p, uni(seq_len(p, b0, over))) == 1);
    if (ALONE || wave == 0) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
            if (valid[k]) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    put_row<TQ, D>(p, whole, PRE ? p.nchunk + part : part, sb[k], h, si[k], 16 * d + 4 * g, acc[k][d], m[k], l[k]);
            }
    }
    if constexpr (PRE) {
        if (wave == 0) {
            stores_done();
            if (lane == 0) sh.done[0] = last_of_tile<ROWS>(p, h, tile);
        }
        __syncthreads();
        const int64_t c0 = (int64_t)tile * ROWS;
        if (sh.done[0]) join_rows<TQ, D, 64 * NW>(p, h, c0, (int)min((int64_t)ROWS, rows - c0), sh.join);
    } else {
        if (!whole) own_done<TQ, D>(p, ALONE || wave == 0, b0, h, sh);
    }
}

template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_or_0(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_sum_i(int x) {
    x += dpp_or_0<0x111, 0xf>(x);
    x += dpp_or_0<0x112, 0xf>(x);
    x += dpp_or_0<0x114, 0xf>(x);
    x += dpp_or_0<0x118, 0xf>(x);
    x += dpp_or_0<0x142, 0xa>(x);
    x += dpp_or_0<0x143, 0xc>(x);
    return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int pages_at(const AttendParams &p, int b) {
    bool over = false;
    return b < p.B ? (seq_len(p, b, over) + PG - 1) / PG : 0;
}
// Parts of all sequences (`units` workgroups take each: heads and row tiles) for parts of c pages.
__device__ __forceinline__ int parts_in_all(const AttendParams &p, int first, int c) {
    int n = 0;
    for (int b = thread_x() % 64; b < p.B; b += 64) {
        const int q = b < 64 ? first : pages_at(p, b);
        n += max((q + c - 1) / c, 1);
    }
    return wave_sum_i(n);
}
// Pages of a part, the same for every sequence: only the device knows the lengths, so every wave works it out for itself.
// Never more than p.nchunk parts of a sequence, which is what the workspace holds.  `first`: pages of sequence lane.
//   One part, if no sequence has more than two times p.least: the second step costs less than the join (B4 H12 D64 L1500 e4m3:
//   9.9 us, 13.7 in two parts).
//   Else the least multiple of p.least for which all parts run at once, p.slots workgroups (B16 H12 D64 L2048 fp16: 22.7 us; 43.8 where
//   that was given up for 24 pages or more, 35 with two workgroups a CU).
//   Where that takes SHORT_PART pages or more: parts for one workgroup a CU if they come out even (at most an eighth above the
//   CU's share of the pages), else for two, else for four (B4 H12 D64 L65536 e4m3: 84.5, 86.9, 88.9 us; B16 H12, ragged to 20000:
//   80, 65.0, 65.5).
__device__ __forceinline__ int part_pages(const AttendParams &p, int first, int64_t units, int most) {
    int64_t work = 0;
    int longest = 0;
    for (int b = thread_x() % 64; b < p.B; b += 64) {
        const int q = b < 64 ? first : pages_at(p, b);
        work += q;
        longest = max(longest, q);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) work += __shfl_xor(work, o, 64);
    work *= units;
    const int floor = max(p.least, (p.P + p.nchunk - 1) / p.nchunk);
    if (p.npchunk == 0 && !__any(longest > 2 * p.least)) return max(2 * p.least, floor);
    int c = max((int)min((work + p.slots - 1) / p.slots + p.least - 1, (int64_t)SHORT_PART) / p.least * p.least, floor);
    for (int k = 0; k < 10 && c < SHORT_PART && p.B * units < p.slots; ++k) {
        if (parts_in_all(p, first, c) * units <= p.slots) return c;
        c = (c + c / 8 + p.least) / p.least * p.least;
    }
    for (int r = 1; r <= ROUNDS; r *= 2) {
        c = (int)min((int64_t)most, max((int64_t)max(LONG_PART, floor), (work + r * CUS - 1) / (r * CUS)));
        for (int k = 0; k < 4 && c < most; ++k) {
            if (parts_in_all(p, first, c) * units <= r * CUS) return c;
            if (k < 3) c = min(c + (c + 23) / 24, most);
        }
    }
    return max(c, floor);
}

// KIND 1, 4: own rows by the few form with that many; 0: by the wide form.  NC: 16-row sets of the prefix's tiles (0: no prefix).
// ALONE: every wave takes a sequence's own rows of one head by itself.
template <typename TQ, typename TS, int D, int KIND, int NC, bool ALONE>
__global__ __launch_bounds__(64 * waves(D)) void fpa_attend_kernel(AttendParams p) {
    constexpr int NW = waves(D);
    __shared__ __align__(16) Shared<D, (NC ? NC : 1)> sh;
    __shared__ __align__(16) TQ weights[KIND ? NW : 1][KIND ? KIND * PG : 1];
    int64_t id = group_x();
    const int H = p.c.H, nrt = (p.N + CW - 1) / CW;  // tiles of a sequence's rows
    const int lane = thread_x() % 64, units = H * nrt;
    int first = 0;
    if constexpr (!ALONE) {
        if (p.nchunk > 1) {
            first = pages_at(p, lane);
            p.chunk = uni(part_pages(p, first, units, most_pages(D)));
        }
    }
    if constexpr (NC > 0) {
        constexpr int ROWS = tile_rows<NC>();
        const int tiles = (int)(((int64_t)p.B * p.N + ROWS - 1) / ROWS);
        // Tiles of the same pages run on one XCD (workgroups go to the eight in turn), one after the other, so that its L2 has
        // what the first of them read.
        const int64_t units = (int64_t)p.npchunk * H, npre = (units + 7) / 8 * 8 * tiles;
        if (id < npre) {
            const int64_t unit = id / (8 * tiles) * 8 + id % 8;
            if (unit < units)
                wide_rows<TQ, TS, D, NC, true, false>(p, 0, (int)(unit / p.npchunk), (int)(id / 8 % tiles), (int)(unit % p.npchunk), sh);
            return;
        }
        id -= npre;
    }
    if constexpr (ALONE) {
        id = id * NW + uni(thread_x() / 64);
        if (id >= (int64_t)p.B * H * nrt) {
            if (p.npchunk > 0) own_done<TQ, D>(p, false, 0, 0, sh);  // the others' barriers
            return;
        }
        // waves of a workgroup: one head, the same tiles
        const int tile = (int)(id % nrt), h = (int)(id / nrt / p.B), b = (int)(id / nrt % p.B);
        if constexpr (KIND > 0)
            few_rows<TQ, TS, D, KIND, true>(p, b, h, 0, sh, weights);
        else
            wide_rows<TQ, TS, D, 1, false, true>(p, b, h, tile, 0, sh);
    } else {
        // item j = id / units of the sequences' parts in a row
        int j = (int)(id / units), b = p.nchunk > 1 ? -1 : j, part = 0;
        for (int b0 = 0; b0 < p.B && p.nchunk > 1; b0 += 64) {
            const int q = b0 == 0 ? first : pages_at(p, b0 + lane);
            int n = b0 + lane < p.B ? max((q + p.chunk - 1) / p.chunk, 1) : 0;
            const int mine = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int u = __shfl_up(n, o, 64);
                if (lane >= o) n += u;
            }
            const uint64_t behind = __ballot(n > j);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                b = b0 + l;
                part = uni(j - __shfl(n - mine, l, 64));
                break;
            }
            j -= __builtin_amdgcn_readlane(n, 63);
        }
        if (b < 0) return;
        const int h = (int)(id % units) / nrt, tile = (int)(id % units) % nrt;
        if constexpr (KIND > 0)
            few_rows<TQ, TS, D, KIND, false>(p, b, h, part, sh, weights);
        else
            wide_rows<TQ, TS, D, 1, false, false>(p, b, h, tile, part, sh);
    }
}

// Row tiles of the prefix: 32 rows where there are more than 16 and their accumulators fit (fp16 to D = 128, fp32 to 64).
constexpr bool two_sets(int D, bool f32) { return D <= (f32 ? 64 : 128); }
int prefix_sets(int D, int64_t rows, bool f32) { return rows > CW && two_sets(D, f32) ? 2 : 1; }

// Steps a page of the kernels' forms: kind and nc as the kernel's, nc > 0: of the prefix's part.
template <typename TQ, typename TS, int D> int steps_of_d(int kind, int nc) {
    if (nc == 2) return PG / wide_keys<TQ, TS, D, 2>();
    if (nc == 1 || kind == 0) return PG / wide_keys<TQ, TS, D, 1>();
    return PG / (kind == 1 ? few_keys<TQ, TS, D, 1>() : few_keys<TQ, TS, D, 4>());
}
template <typename TQ, typename TS> int steps_of(int D, int kind, int nc) {
    switch (D) {
        case 16: return steps_of_d<TQ, TS, 16>(kind, nc);
        case 32: return steps_of_d<TQ, TS, 32>(kind, nc);
        case 64: return steps_of_d<TQ, TS, 64>(kind, nc);
        case 128: return steps_of_d<TQ, TS, 128>(kind, nc);
        case 256: return steps_of_d<TQ, TS, 256>(kind, nc);
    }
    return 1;
}

// Where a wave takes a sequence alone there are many of them with few rows each: those kernels are built for N <= 4, and behind
// a prefix for its tiles of 32 rows.
constexpr bool alone_built(int kind, int nc) { return kind > 0 && nc != 1; }

template <typename TQ, typename TS, int D, int KIND, int NC> void launch_attend_k(const AttendParams &p, hipStream_t s) {
    constexpr int NW = waves(D), ROWS = tile_rows<(NC ? NC : 1)>();
    const int64_t rows = (int64_t)p.B * p.N, H = p.c.H, own = (int64_t)p.B * H * ((p.N + CW - 1) / CW);
    const int64_t pre = NC ? (p.npchunk * H + 7) / 8 * 8 * ((rows + ROWS - 1) / ROWS) : 0;
    if constexpr (alone_built(KIND, NC))
        if (p.alone) {
            hipLaunchKernelGGL((fpa_attend_kernel<TQ, TS, D, KIND, NC, true>), dim3((uint32_t)(pre + (own + NW - 1) / NW)), dim3(64 * NW), 0, s, p);
            return;
        }
    hipLaunchKernelGGL((fpa_attend_kernel<TQ, TS, D, KIND, NC, false>), dim3((uint32_t)(pre + p.own_groups)), dim3(64 * NW), 0, s, p);
}

template <typename TQ, typename TS, int D> hipError_t launch_attend_d(const AttendParams &p, hipStream_t s) {
    constexpr bool TWO = two_sets(D, sizeof(TQ) == 4);
    if (p.npchunk == 0) {
        if (p.N == 1)
            launch_attend_k<TQ, TS, D, 1, 0>(p, s);
        else if (p.N <= 4)
            launch_attend_k<TQ, TS, D, 4, 0>(p, s);
        else
            launch_attend_k<TQ, TS, D, 0, 0>(p, s);
    } else if (TWO && p.B * (int64_t)p.N > CW) {
        if (p.N <= 4)
            launch_attend_k<TQ, TS, D, 4, TWO ? 2 : 1>(p, s);
        else
            launch_attend_k<TQ, TS, D, 0, TWO ? 2 : 1>(p, s);
    } else {
        if (p.N <= 4)
            launch_attend_k<TQ, TS, D, 4, 1>(p, s);
        else
            launch_attend_k<TQ, TS, D, 0, 1>(p, s);
    }
    return hipGetLastError();
}

}  // namespace

// Head sizes to 64, and above: each pair of types and half is a file of its own, which compile side by side.
template <typename TQ, typename TS> hipError_t launch_attend_small(const AttendParams &p, int D, hipStream_t s) {
    switch (D) {
        case 16: return launch_attend_d<TQ, TS, 16>(p, s);
        case 32: return launch_attend_d<TQ, TS, 32>(p, s);
        case 64: return launch_attend_d<TQ, TS, 64>(p, s);
    }
    return hipErrorInvalidValue;
}
template <typename TQ, typename TS> hipError_t launch_attend_large(const AttendParams &p, int D, hipStream_t s) {
    switch (D) {
        case 128: return launch_attend_d<TQ, TS, 128>(p, s);
        case 256: return launch_attend_d<TQ, TS, 256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace fpa
