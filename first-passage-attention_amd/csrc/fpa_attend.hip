// fpa_attend.hip -- First Passage Attention of new tokens against a paged cache.
//
// Query i of N stands at position t = len - N + i of its sequence and attends to the keys s <= t:
//   o_t = sum_s softmax_s(q_t . k_s / sqrt(D) + beta min(0, X_ts - psi_s)) v_s,   X_ts = min_{s < u <= t} phi_u
// (X_tt is +inf).  A shared prefix of PL positions comes before the sequence's own position 0: for its keys
//   X_ts = min(min_{s < u < PL} phi_u, min_{0 <= u <= t} phi_u of the sequence itself),
// so that only the second term differs between the requests, and the rows of all of them form one product
// with the prefix's K and V.
//
// One wave takes 64 keys (a page) at a time for 16 query rows, on the 16x16 MFMA: S^T = K Q^T, then
// O^T += V^T P^T.  Both cache operands go from HBM straight into registers: the pages hold K by rows and V
// transposed, and the key of score register (a, j) of lane group g is 16 g + 4 a + j, so that a lane's 16
// probabilities belong to 16 consecutive keys: as they stand they are the B operand of the second product, whose
// A operand is 16 consecutive values of a V^T row, and the range minimum is a scan inside the lane.
//
// The pages are taken from the last to the first and the running minimum is carried along; what lies
// between a wave's pages and its queries is one phi_min value a page.  A sequence is cut into parts of whole
// pages that run side by side (each wave of a workgroup takes a quarter of its part); a merge kernel joins
// them in a fixed order.
//
// Softmax statistics and O are fp32.  P is rounded to fp16 for fp16 queries (at most 1, so what is lost is
// below 2^-25 of the row's largest weight); fp32 queries keep fp32 throughout.  With e4m3 pages the row's
// power of two of V goes into the logit: the weights w_s = p_s 2^e_s are what multiplies the codes, the running
// maximum is that of w, so that w fills fp16's range whatever the scales are, and the sum takes w_s 2^-e_s.
//
// What a query must not see is never multiplied: masked scores are replaced, V rows behind the sequence's end
// are cleared, and an infinity or NaN in a V row that only some of the 16 queries see is left out of the product and
// added for those alone.
#include <type_traits>

#include "fpa_common.h"
#include "fpa_serve.h"

namespace fpa {

namespace {

constexpr int CW = 16;  // query rows of a wave
constexpr int NWV = 4;  // waves of a workgroup

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// N consecutive cache values of a lane, first as loaded, then as matrix operands.
template <typename TS, int N> struct Raw {
    static constexpr int BYTES = N * (int)sizeof(TS);
    static_assert(BYTES % 4 == 0, "whole words");
    uint32_t w[BYTES / 4];
    __device__ __forceinline__ void load(const TS *p) {
        const char *b = reinterpret_cast<const char *>(p);
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(b + 16 * i);
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
// Clears the values of a run from element `n` on and those that are not finite; true if there were such before n.
template <typename TS, int N> __device__ __forceinline__ bool clean(Raw<TS, N> &r, int n) {
    constexpr int PW = 4 / sizeof(TS), BITS = 8 * sizeof(TS);  // values of a word
    constexpr uint32_t ONE = BITS == 32 ? 0xffffffffu : (1u << (BITS % 32)) - 1;
    bool some = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int sh = i % PW * BITS;
        const bool off = beyond_bits<TS>(r.w[i / PW] >> sh & ONE);
        if (i >= n || off) r.w[i / PW] &= ~(ONE << sh);
        some |= i < n && off;
    }
    return some;
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

__device__ __forceinline__ float from_group(float x, int lane, int d) { return __shfl(x, (lane + 16 * d) & 63, 64); }
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

constexpr uint32_t BAD = 0xbf800000u;  // -1.0f in place of a row's sum: its table names no page, or its length passes the table
// NaN that the compiler does not see as one (it may drop what it can tell to be NaN).
__device__ __forceinline__ float quiet_nan() {
    uint32_t b = 0x7fc00000u;
    asm("" : "+v"(b));
    return __uint_as_float(b);
}

// Length of sequence b, at most what its table holds.
__device__ __forceinline__ int seq_len(const AttendParams &p, int b, bool &bad) {
    const int L = p.lengths[b];
    const int64_t cap = (int64_t)p.P * PG;
    if (L > cap) bad = true;
    return L < 0 ? 0 : (L > cap ? (int)cap : L);
}

template <typename TQ, typename TS, int D>
__global__ __launch_bounds__(64 * NWV) void fpa_attend_kernel(AttendParams p) {
    typedef typename Quad<TQ>::t quad_t;
    constexpr int DG = D / 4;   // features of a lane group in the score product
    constexpr int ND = D / 16;  // feature tiles of the output
    extern __shared__ __align__(16) float smem[];
    const int lane = thread_x() % 64, wave = uni(thread_x() / 64), c = lane % 16, g = lane / 16;
    const int H = p.c.H;

    // Which rows, and which pages.
    const int nct = (int)(((int64_t)p.B * p.N + CW - 1) / CW);  // row tiles of the prefix: over all sequences
    const int nrt = (p.N + CW - 1) / CW;                        // of one sequence
    const int64_t npre = (int64_t)p.npchunk * H * nct;
    int64_t id = group_x();
    const bool pre = id < npre;
    int h, b, i, part;           // this lane's column: sequence b, query i
    int ps, npg, pf;             // first page of the part, pages of the segment, pages that every row sees whole
    int pe;                      // page behind the part
    int last;                    // last position of the segment that the lane's row sees, -1: none
    int lmax;                    // the largest `last`
    const int32_t *table;
    bool valid, bad = false;     // bad: of this lane's row
    bool missing = false;        // a page of the segment that its table does not name: every row's
    float x0 = pinf();           // min of phi from the segment's end to the row's own position
    if (pre) {
        const int ct = (int)(id % nct);
        id /= nct;
        part = (int)(id % p.npchunk);
        h = (int)(id / p.npchunk);
        const int64_t col = (int64_t)ct * CW + c;
        valid = col < (int64_t)p.B * p.N;
        b = valid ? (int)(col / p.N) : 0;
        i = valid ? (int)(col % p.N) : 0;
        table = p.prefix;
        npg = (p.PL + PG - 1) / PG;
        pf = p.PL / PG;
        ps = part * p.pchunk;
        pe = min(ps + p.pchunk, npg);
        lmax = p.PL - 1;
        const int t = seq_len(p, b, bad) - p.N + i;
        last = valid && t >= 0 ? lmax : -1;
        // min of the sequence's own phi up to t, the lane groups taking the whole pages in turn
        const int32_t *tb = p.table + (int64_t)b * p.stable;
        const int full = (t + 1) / PG;  // t >= -N: C++ division towards 0 gives at most 0 for t < 0
        for (int k = g; k < full; k += 4) {
            const int page = tb[k];
            if ((uint32_t)page >= (uint64_t)p.c.n)
                bad = true;
            else
                x0 = fminf(x0, p.c.phi_min[(int64_t)page * H + h]);
        }
        const int rest = t >= 0 ? (t + 1) % PG : 0;
        if (rest > 0) {
            const int page = tb[full];
            if ((uint32_t)page >= (uint64_t)p.c.n) {
                bad = true;
            } else {
                const float *ph = p.c.phi + ((int64_t)page * H + h) * PG;
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (16 * g + k < rest) x0 = fminf(x0, ph[16 * g + k]);
            }
        }
        x0 = min_groups(x0);
    } else {
        id -= npre;
        const int rt = (int)(id % nrt);
        id /= nrt;
        const int bh = (int)(id % ((int64_t)p.B * H));
        part = (int)(id / ((int64_t)p.B * H));
        b = bh / H;
        h = bh % H;
        i = rt * CW + c;
        valid = i < p.N;
        if (!valid) i = 0;
        table = p.table + (int64_t)b * p.stable;
        const int L = uni(seq_len(p, b, bad));
        const int tmin = L - p.N + rt * CW;
        lmax = min(tmin + CW, L) - 1;
        const int t = tmin + c;
        last = valid && t >= 0 ? t : -1;
        npg = lmax >= 0 ? lmax / PG + 1 : 0;
        pf = tmin >= 0 ? (tmin + 1) / PG : 0;
        ps = part * p.chunk;
        pe = min(ps + p.chunk, npg);
        // Parts behind the sequence's end: nothing reads their results.
        if (part > 0 && ps >= (L + PG - 1) / PG) return;
    }

    // The lane's query row.
    quad_t qv[DG / 4];
    if (valid) {
        Raw<TQ, DG> r;
        r.load(static_cast<const TQ *>(p.q) + (int64_t)b * p.sq.b + (int64_t)h * p.sq.h + (int64_t)i * p.sq.t + g * DG);
#pragma unroll
        for (int k = 0; k < DG / 4; ++k) qv[k] = quad<TQ>(r, k);
    } else {
#pragma unroll
        for (int k = 0; k < DG / 4; ++k) qv[k] = quad_t{0, 0, 0, 0};
    }
    const float beta2 = p.beta[h] * LOG2E;

    // The wave's pages [ws, we), and the minimum of phi behind them.
    const int per = pe > ps ? (pe - ps + NWV - 1) / NWV : 0;
    const int ws = ps + wave * per, we = min(ws + per, pe);
    float carry = x0;
    if (ws < we) {
        float m = pinf();
        for (int k = we + lane; k < pf; k += 64) {
            const int page = table[k];
            if ((uint32_t)page >= (uint64_t)p.c.n)
                missing = true;
            else
                m = fminf(m, p.c.phi_min[(int64_t)page * H + h]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fminf(m, __shfl_xor(m, o, 64));
        for (int k = max(we, pf); k < npg; ++k) {  // at most two pages that some rows see in part
            const int page = table[k];
            if ((uint32_t)page >= (uint64_t)p.c.n) {
                missing = true;
                continue;
            }
            const float *ph = p.c.phi + ((int64_t)page * H + h) * PG + 16 * g;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (k * PG + 16 * g + e <= last) m = fminf(m, ph[e]);
        }
        carry = fminf(carry, min_groups(m));
    }

    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = ninf(), l = 0.f;

    auto page_step = [&](auto tail_tag, int pg, int64_t ph) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail_tag)::value;
        const TS *kp = static_cast<const TS *>(p.c.k) + ph * PG * D;
        const TS *vp = static_cast<const TS *>(p.c.v) + ph * PG * D;
        // S^T: score (a, j) of the lane is key 16 g + 4 a + j
        float t[16];
        {
            f32x4 phv[4], psv[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                phv[a] = *reinterpret_cast<const f32x4 *>(p.c.phi + ph * PG + 16 * g + 4 * a);
                psv[a] = *reinterpret_cast<const f32x4 *>(p.c.psi + ph * PG + 16 * g + 4 * a);
            }
            u32x4 kew;
            if constexpr (sizeof(TS) == 1) kew = *reinterpret_cast<const u32x4 *>(p.c.k_exp + ph * PG + 16 * g);
            const int key0 = pg * PG + 16 * g;
            // range minima of the lane's keys, last to first
            float x[16], r = pinf();
#pragma unroll
            for (int e = 15; e >= 0; --e) {
                x[e] = r;
                const float f = phv[e / 4][e % 4];
                r = fminf(r, (!TAIL || key0 + e <= last) ? f : pinf());
            }
            const float r1 = from_group(r, lane, 1), r2 = from_group(r, lane, 2), r3 = from_group(r, lane, 3);
            float behind = carry;
            if (g < 3) behind = fminf(behind, r1);
            if (g < 2) behind = fminf(behind, r2);
            if (g < 1) behind = fminf(behind, r3);
            carry = fminf(fminf(carry, r), fminf(r1, fminf(r2, r3)));
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                Raw<TS, DG> kr;
                kr.load(kp + (16 * (c / 4) + 4 * a + c % 4) * D + g * DG);
                quad_t kq[DG / 4];
#pragma unroll
                for (int k = 0; k < DG / 4; ++k) kq[k] = quad<TQ>(kr, k);
                const f32x4 s = mma<DG / 4>(kq, qv, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 4 * a + j;
                    float sc = p.sc2;
                    if constexpr (sizeof(TS) == 1) sc *= pow2((int)(int8_t)(kew[a] >> (8 * j)));
                    const float bias = beta2 * fminf(fminf(x[e], behind) - psv[a][j], 0.f);
                    t[e] = s[j] * sc + bias;
                    if (TAIL && key0 + e > last) t[e] = ninf();
                }
            }
        }
        u32x4 vew;
        if constexpr (sizeof(TS) == 1) {
            vew = *reinterpret_cast<const u32x4 *>(p.c.v_exp + ph * PG + 16 * g);
#pragma unroll
            for (int e = 0; e < 16; ++e) t[e] += (float)(int8_t)(vew[e / 4] >> (8 * (e % 4)));
        }
        float mt = t[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mt = fmaxf(mt, t[e]);
        const float mn = fmaxf(m, max_groups(mt));
        const float ref = mn == ninf() ? 0.f : mn;
        const float alpha = fexp2(m - ref);
        m = mn;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            t[e] = fexp2(t[e] - ref);
            if constexpr (sizeof(TS) == 1)
                sum += t[e] * pow2(-(int)(int8_t)(vew[e / 4] >> (8 * (e % 4))));
            else
                sum += t[e];
        }
        l = l * alpha + sum;
        quad_t pq[4];
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) pq[a][j] = (TQ)t[4 * a + j];
        bool some = false;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            Raw<TS, 16> vr;
            vr.load(vp + (16 * d + c) * PG + 16 * g);
            if constexpr (TAIL) some |= clean(vr, lmax + 1 - pg * PG - 16 * g);
            quad_t vq[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) vq[a] = quad<TQ>(vr, a);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[d][j] *= alpha;
            acc[d] = mma<4>(vq, pq, acc[d]);
        }
        if (TAIL && __any(some)) {  // infinities and NaN, for the rows that see them
            for (int e = 0; e < PG; ++e) {
                float w = t[0];
#pragma unroll
                for (int k = 1; k < 16; ++k) w = e % 16 == k ? t[k] : w;
                w = __shfl(w, e / 16 * 16 + c, 64);
                const bool sees = pg * PG + e <= last;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const TS *vx = vp + (16 * d + 4 * g + j) * PG + e;
                        uint32_t bits;
                        float x;
                        if constexpr (sizeof(TS) == 1) {
                            bits = vx->code;
                            x = quiet_nan();
                        } else if constexpr (sizeof(TS) == 2) {
                            bits = *reinterpret_cast<const uint16_t *>(vx);
                            x = (float)*vx;
                        } else {
                            bits = *reinterpret_cast<const uint32_t *>(vx);
                            x = *vx;
                        }
                        if (sees && beyond_bits<TS>(bits)) acc[d][j] += w * x;
                    }
            }
        }
    };
    for (int pg = we - 1; pg >= ws; --pg) {
        const int page = uni(table[pg]);
        if ((uint32_t)page >= (uint64_t)p.c.n) {
            missing = true;
            continue;
        }
        const int64_t ph = (int64_t)page * H + h;
        if (pg >= pf)
            page_step(std::true_type{}, pg, ph);
        else
            page_step(std::false_type{}, pg, ph);
    }

    // The waves' results together, in order.  smem: [wave][row] maximum and sum, then [wave][row][D].
    l = sum_groups(l);
    if (last < 0) {  // a row that sees nothing: the prefix's whole pages are not masked for it
        m = ninf();
        l = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (__any(missing) || max_groups(bad ? 1.f : 0.f) > 0.f) l = __uint_as_float(BAD);
    const int rows = (int)min((int64_t)CW, pre ? (int64_t)p.B * p.N : (int64_t)p.N);  // rows kept in smem
    float *ml = smem, *so = smem + 2 * NWV * CW;
    if (g == 0) {
        ml[2 * (wave * CW + c)] = m;
        ml[2 * (wave * CW + c) + 1] = l;
    }
    if (c < rows) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
            *reinterpret_cast<f32x4 *>(so + ((int64_t)wave * rows + c) * D + 16 * d + 4 * g) = acc[d];
    }
    __syncthreads();
    const bool whole = p.nchunk <= 1 && p.npchunk == 0;  // this part is all: write the output itself
    const int64_t R = (int64_t)p.B * H * p.N;
    for (int e = thread_x(); e < rows * D; e += 64 * NWV) {
        const int r = e / D, d = e % D;
        // the row's sequence and query, as lane r of the waves has them
        int rb, ri;
        if (pre) {
            const int64_t col = (int64_t)((int64_t)group_x() % nct) * CW + r;
            if (col >= (int64_t)p.B * p.N) break;
            rb = (int)(col / p.N);
            ri = (int)(col % p.N);
        } else {
            rb = b;
            ri = (int)(((int64_t)group_x() - npre) % nrt) * CW + r;
            if (ri >= p.N) break;
        }
        float mm = ninf();
        bool rbad = false;
#pragma unroll
        for (int w = 0; w < NWV; ++w) {
            mm = fmaxf(mm, ml[2 * (w * CW + r)]);
            rbad |= __float_as_uint(ml[2 * (w * CW + r) + 1]) == BAD;
        }
        const float ref = mm == ninf() ? 0.f : mm;
        float ll = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < NWV; ++w) {
            const float a = fexp2(ml[2 * (w * CW + r)] - ref);
            ll += a * ml[2 * (w * CW + r) + 1];
            x += a * so[((int64_t)w * rows + r) * D + d];
        }
        if (rbad) ll = __uint_as_float(BAD);
        const int64_t row = ((int64_t)rb * H + h) * p.N + ri;
        if (whole) {
            const bool none = (__float_as_uint(ll) << 1) == 0;
            x = rbad ? quiet_nan() : none ? 0.f : x / ll;
            static_cast<TQ *>(p.o)[(int64_t)rb * p.so.b + (int64_t)h * p.so.h + (int64_t)ri * p.so.t + d] = (TQ)x;
        } else {
            const int64_t slot = (int64_t)(pre ? p.nchunk + part : part) * R + row;
            p.part[slot * D + d] = x;
            if (d == 0) {
                p.ml[2 * slot] = mm;
                p.ml[2 * slot + 1] = ll;
            }
        }
    }
}

// Joins the parts of each row in order; one thread per feature.
template <typename TQ, int D> __global__ __launch_bounds__(256) void fpa_attend_merge_kernel(AttendParams p) {
    const int H = p.c.H;
    const int64_t R = (int64_t)p.B * H * p.N, e = (int64_t)group_x() * 256 + thread_x();
    const int64_t row = e / D;
    const int d = (int)(e % D);
    if (row >= R) return;
    const int i = (int)(row % p.N), h = (int)(row / p.N % H), b = (int)(row / p.N / H);
    bool bad = false;
    const int L = seq_len(p, b, bad);
    const int own = ((L + PG - 1) / PG + p.chunk - 1) / p.chunk;
    const int parts = own + p.npchunk;
    float m = ninf(), l = 0.f, x = 0.f;
    for (int k = 0; k < parts; ++k) {
        const int64_t slot = (int64_t)(k < own ? k : p.nchunk + k - own) * R + row;
        const float mk = p.ml[2 * slot], lk = p.ml[2 * slot + 1];
        if (__float_as_uint(lk) == BAD) bad = true;
        const float mn = fmaxf(m, mk), ref = mn == ninf() ? 0.f : mn;
        const float a = fexp2(m - ref), w = fexp2(mk - ref);
        l = l * a + lk * w;
        x = x * a + p.part[slot * D + d] * w;
        m = mn;
    }
    const bool none = (__float_as_uint(l) << 1) == 0;
    x = bad ? quiet_nan() : none ? 0.f : x / l;
    static_cast<TQ *>(p.o)[(int64_t)b * p.so.b + (int64_t)h * p.so.h + (int64_t)i * p.so.t + d] = (TQ)x;
}

template <typename TQ, typename TS, int D> hipError_t launch_attend_d(const AttendParams &p, hipStream_t s) {
    const int64_t rows = (int64_t)p.B * p.N, H = p.c.H;
    const int64_t pre = (int64_t)p.npchunk * H * ((rows + CW - 1) / CW);
    const int64_t own = (int64_t)p.nchunk * p.B * H * ((p.N + CW - 1) / CW);
    const int64_t kept = p.npchunk ? (rows < CW ? rows : CW) : (p.N < CW ? p.N : CW);
    const size_t lds = (size_t)(2 * NWV * CW + NWV * kept * D) * 4;
    hipLaunchKernelGGL((fpa_attend_kernel<TQ, TS, D>), dim3((uint32_t)(pre + own)), dim3(64 * NWV), lds, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || (p.nchunk <= 1 && p.npchunk == 0)) return e;
    hipLaunchKernelGGL((fpa_attend_merge_kernel<TQ, D>), dim3((uint32_t)((rows * H * D + 255) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <typename TQ, typename TS> hipError_t launch_attend_t(const AttendParams &p, int D, hipStream_t s) {
    switch (D) {
        case 16: return launch_attend_d<TQ, TS, 16>(p, s);
        case 32: return launch_attend_d<TQ, TS, 32>(p, s);
        case 64: return launch_attend_d<TQ, TS, 64>(p, s);
        case 128: return launch_attend_d<TQ, TS, 128>(p, s);
        case 256: return launch_attend_d<TQ, TS, 256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attend(const AttendParams &p, int dtype, int store, int D, hipStream_t s) {
    if (dtype == ST_F16 && store == ST_F16) return launch_attend_t<f16, f16>(p, D, s);
    if (dtype == ST_F32 && store == ST_F32) return launch_attend_t<float, float>(p, D, s);
    if (dtype == ST_F16 && store == ST_E4M3) return launch_attend_t<f16, e4m3>(p, D, s);
    if (dtype == ST_F32 && store == ST_E4M3) return launch_attend_t<float, e4m3>(p, D, s);
    return hipErrorInvalidValue;
}

void attend_parts(int64_t items, int64_t pages, int &chunk, int &nchunk) {
    // Parts of at least NWV pages (one a wave), and about 1024 workgroups (four on a CU).
    int64_t want = items >= 1024 ? 1 : (1024 + items - 1) / items;
    int64_t c = (pages + want - 1) / want;
    c = c < NWV ? NWV : c;
    c = c > 128 ? 128 : c;  // long sequences among short ones are spread in any case
    chunk = (int)c;
    nchunk = (int)((pages + c - 1) / c);
}

}  // namespace fpa
