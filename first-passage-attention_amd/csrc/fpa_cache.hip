// fpa_cache.hip -- writing positions into the pages of a cache and reading them back.
//
// e4m3 rows.  The row of K or V of one position and head is kept as code * 2^e with
//   e = clamp(ceil(log2(max |x| / 448)), -60, 60)   (-60 for a row of zeros),   code = e4m3(x * 2^-e),
// rounded to nearest even, saturating.  A power of two costs an 8-bit floating-point format nothing (its
// relative step is the same in every binade; only values 2^-15 below the row's maximum reach its subnormals),
// scaling by it is exact, so the code is one rounding of the value itself, and the products take it out again
// exactly: for K on the score, for V as an addition to the logit.  NaN stays NaN, an infinity saturates.
//
// Both kernels are passes over their bytes: one workgroup per (page, head, sequence), K rows moved in 16-byte
// pieces, V turned in LDS (its rows a few bytes apart from a power of two, so that columns lie in different banks).  Prompts, B8
// H12 D64 to 2048 positions, fp16 to e4m3: append 14 us, read 10 to 12, 39 MB each (2.8 and 3.5 TB/s; the turn in LDS and the start
// of 3168 workgroups with few bytes each are what keeps them from the copy's 5.2).  One token of B64: 5.9 and 3.9 us, launch
// and a chain of table, row and store.
#include "fpa_common.h"
#include "fpa_serve.h"

namespace fpa {

namespace {

// Exponent of a row whose largest magnitude is amax (not NaN): amax = m 2^x with m in [0.5, 1) is at most
// 448 * 2^e = 0.875 * 2^(9 + e) for e = x - 9 if m <= 0.875, else e = x - 8.  Subnormal amax: -60 either way.
__device__ __forceinline__ int row_exp(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 126;
    const int e = (b & 0x7fffffu) > 0x600000u ? x - 8 : x - 9;
    return max(EXP_MIN, min(EXP_MAX, e));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ bool is_nan(float x) { return (__float_as_uint(x) & 0x7fffffffu) > 0x7f800000u; }
// |x| with NaN as 0.
__device__ __forceinline__ float mag(float x) { return is_nan(x) ? 0.f : __uint_as_float(__float_as_uint(x) & 0x7fffffffu); }

// Four scaled values as e4m3 codes.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    float x[4] = {a, b, c, d};
    uint32_t nan = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        nan |= is_nan(x[i]) ? 0x7fu << (8 * i) : 0u;
        x[i] = __builtin_amdgcn_fmed3f(x[i], -448.f, 448.f);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
    return (uint32_t)w | nan;
}

// A lane's 16 bytes of one input row.
template <typename TX> struct Piece {
    static constexpr int N = 16 / sizeof(TX);
    float x[N];
    __device__ __forceinline__ void load(const TX *p) {
        if constexpr (sizeof(TX) == 2) {
            const h8 v = *reinterpret_cast<const h8 *>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
        } else {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = v[i];
        }
    }
    // as the N values of the cache at dst
    __device__ __forceinline__ void store(f16 *dst) const {
        h8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (f16)x[i % N];
        *reinterpret_cast<h8 *>(dst) = v;
    }
    __device__ __forceinline__ void store(float *dst) const { *reinterpret_cast<f32x4 *>(dst) = f32x4{x[0], x[1], x[2], x[3]}; }
    __device__ __forceinline__ void store(e4m3 *dst) const {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            reinterpret_cast<uint32_t *>(dst)[i / 4] = codes4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
    // Scales the row that LPR neighbouring lanes hold together for e4m3; returns its exponent.
    template <int LPR> __device__ __forceinline__ int scale() {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, mag(x[i]));
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const int e = row_exp(m);
        const float s = pow2(-e);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= s;
        return e;
    }
};

template <typename TX, typename TS, int D>
__global__ __launch_bounds__(256) void fpa_append_kernel(MoveParams p) {
    constexpr int N16 = Piece<TX>::N, LPR = D / N16, RPP = 256 / LPR;  // lanes of a row, rows of a pass
    constexpr int LP = D + (sizeof(TS) == 1 ? 4 : 16 / (int)sizeof(TS));   // pitch of the V tile in LDS
    __shared__ __align__(16) TS tile[PG * LP];
    const int tid = thread_x(), h = group_y(), b = group_z();
    const int64_t start = p.start[b];
    int64_t n = p.counts ? p.counts[b] : p.N;
    n = n > p.N ? p.N : n;
    if (start < 0) return;
    const int64_t pg = start / PG + group_x();  // page of the sequence
    const int lo = group_x() == 0 ? (int)(start % PG) : 0;
    const int64_t left = start + n - pg * PG;  // positions of this page that are written, from its first
    const int hi = left > PG ? PG : (int)left;
    if (left <= lo || pg >= p.P) return;
    const int page = p.table[(int64_t)b * p.stable + pg];
    if ((uint32_t)page >= (uint64_t)p.c.n) return;  // no such page
    const int64_t ph = (int64_t)page * p.c.H + h;
    const int64_t i0 = pg * PG - start;  // token of the page's first position (may be negative)
    const TX *k = static_cast<const TX *>(p.k) + (int64_t)b * p.sk.b + (int64_t)h * p.sk.h;
    const TX *v = static_cast<const TX *>(p.v) + (int64_t)b * p.sv.b + (int64_t)h * p.sv.h;
    TS *ck = static_cast<TS *>(p.c.k) + ph * PG * D;
    TS *cv = static_cast<TS *>(p.c.v) + ph * PG * D;
    const int col = tid % LPR * N16;
    for (int r0 = 0; r0 < PG; r0 += RPP) {
        const int r = r0 + tid / LPR;
        if (r0 + RPP <= lo || r0 >= hi) continue;
        const bool there = r >= lo && r < hi;
        const int rr = min(max(r, lo), hi - 1);  // rows outside read a written one
        Piece<TX> a, c;
        a.load(k + (i0 + rr) * p.sk.t + col);
        c.load(v + (i0 + rr) * p.sv.t + col);
        if constexpr (sizeof(TS) == 1) {
            const int ea = a.template scale<LPR>(), ec = c.template scale<LPR>();
            if (there && tid % LPR == 0) {
                p.c.k_exp[ph * PG + r] = (int8_t)ea;
                p.c.v_exp[ph * PG + r] = (int8_t)ec;
            }
        }
        if (there) {
            a.store(ck + r * D + col);
            c.store(tile + r * LP + col);
        }
    }
    if (tid < PG) {
        const bool there = tid >= lo && tid < hi;
        float x = pinf();
        if (there) {
            x = p.phi[(int64_t)b * p.sphi.b + (int64_t)h * p.sphi.h + (i0 + tid) * p.sphi.t];
            p.c.phi[ph * PG + tid] = x;
            p.c.psi[ph * PG + tid] = p.psi[(int64_t)b * p.spsi.b + (int64_t)h * p.spsi.h + (i0 + tid) * p.spsi.t];
        } else if (tid < lo) {
            x = p.c.phi[ph * PG + tid];
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) x = fminf(x, __shfl_xor(x, o, 64));
        if (tid == 0) p.c.phi_min[ph] = x;
    }
    __syncthreads();
    // V^T: the positions of one feature, in pieces of 16 bytes where the page is written whole.
    constexpr int PC = 16 / sizeof(TS);
    if (lo == 0 && hi == PG) {
        for (int e = tid; e < D * PG / PC; e += 256) {
            const int d = e / (PG / PC), r = e % (PG / PC) * PC;
            uint32_t w[4];
            TS *x = reinterpret_cast<TS *>(w);
#pragma unroll
            for (int i = 0; i < PC; ++i) x[i] = tile[(r + i) * LP + d];
            *reinterpret_cast<u32x4 *>(cv + d * PG + r) = u32x4{w[0], w[1], w[2], w[3]};
        }
    } else {
        const int n = hi - lo;
        for (int e = tid; e < D * n; e += 256) {
            const int d = e / n, r = lo + e % n;
            cv[d * PG + r] = tile[r * LP + d];
        }
    }
}

// N consecutive cache values as float, times the row's power of two.
template <typename TS, int N> __device__ __forceinline__ void values(float (&x)[N], const TS *p, float scale) {
    if constexpr (sizeof(TS) == 1) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const int w = *reinterpret_cast<const int *>(p + i);
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
            x[i] = a[0] * scale;
            x[i + 1] = a[1] * scale;
            x[i + 2] = b[0] * scale;
            x[i + 3] = b[1] * scale;
        }
    } else {
        Piece<TS> q;
        q.load(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = q.x[i];
    }
}

template <typename TX, typename TS, int D>
__global__ __launch_bounds__(256) void fpa_read_kernel(MoveParams p) {
    constexpr int PC = 16 / sizeof(TS);   // positions of a piece of V^T
    constexpr int LP = D + (sizeof(TS) == 1 ? 4 : 16 / (int)sizeof(TS));  // V rows by position in LDS
    constexpr int N16 = Piece<TX>::N, LPR = D / N16;
    __shared__ __align__(16) TS tile[PG * LP];
    const int tid = thread_x(), h = group_y(), b = group_z();
    int64_t start = p.start[b];
    int64_t n = p.counts ? p.counts[b] : p.N;
    n = n > p.N ? p.N : n;
    bool there = start >= 0;
    if (!there) start = 0;  // nothing to read: every row NaN
    const int64_t pg = start / PG + group_x();
    const int lo = group_x() == 0 ? (int)(start % PG) : 0;
    const int64_t left = start + p.N - pg * PG;
    const int hi = left > PG ? PG : (int)left;
    if (left <= lo) return;
    const int64_t i0 = pg * PG - start;
    there = there && pg < p.P;
    const int page = there ? p.table[(int64_t)b * p.stable + pg] : -1;
    there = (uint32_t)page < (uint64_t)p.c.n && page >= 0;
    const int64_t ph = there ? (int64_t)page * p.c.H + h : 0;
    const TS *ck = static_cast<const TS *>(p.c.k) + ph * PG * D;
    const TS *cv = static_cast<const TS *>(p.c.v) + ph * PG * D;
    const int64_t row0 = ((int64_t)b * p.c.H + h) * p.N + i0;
    if (there) {
        if (hi - lo > PG / 4) {  // the page's V, turned
            for (int e = tid; e < D * PG / PC; e += 256) {
                const int d = e / (PG / PC), r = e % (PG / PC) * PC;
                const u32x4 w = *reinterpret_cast<const u32x4 *>(cv + d * PG + r);
                const TS *x = reinterpret_cast<const TS *>(&w);
#pragma unroll
                for (int i = 0; i < PC; ++i) tile[(r + i) * LP + d] = x[i];
            }
        } else {  // a few positions
            const int m = hi - lo;
            for (int e = tid; e < D * m; e += 256) tile[(lo + e % m) * LP + e / m] = cv[e / m * PG + lo + e % m];
        }
    }
    __syncthreads();
    const float nan = __uint_as_float(0x7fc00000u);
    for (int e = lo * LPR + tid; e < hi * LPR; e += 256) {
        const int r = e / LPR, col = e % LPR * N16;
        Piece<TX> k, v;
#pragma unroll
        for (int i = 0; i < N16; ++i) k.x[i] = v.x[i] = i0 + r < n ? nan : 0.f;
        if (there && i0 + r < n) {
            float ks = 1.f, vs = 1.f;
            if constexpr (sizeof(TS) == 1) {
                ks = pow2(p.c.k_exp[ph * PG + r]);
                vs = pow2(p.c.v_exp[ph * PG + r]);
            }
            values<TS, N16>(k.x, ck + r * D + col, ks);
            values<TS, N16>(v.x, tile + r * LP + col, vs);
        }
        k.store(static_cast<TX *>(p.ko) + (row0 + r) * D + col);
        v.store(static_cast<TX *>(p.vo) + (row0 + r) * D + col);
    }
    if (tid >= lo && tid < hi) {
        const bool in = i0 + tid < n;
        p.phio[row0 + tid] = !in ? 0.f : there ? p.c.phi[ph * PG + tid] : nan;
        p.psio[row0 + tid] = !in ? 0.f : there ? p.c.psi[ph * PG + tid] : nan;
    }
}

template <bool READ, typename TX, typename TS, int D> hipError_t launch_move_d(const MoveParams &p, hipStream_t s) {
    const dim3 grid((p.N + PG - 2) / PG + 1, p.c.H, p.B);
    if constexpr (READ)
        hipLaunchKernelGGL((fpa_read_kernel<TX, TS, D>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((fpa_append_kernel<TX, TS, D>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

template <bool READ, typename TX, typename TS> hipError_t launch_move_t(const MoveParams &p, hipStream_t s) {
    switch (p.D) {
        case 16: return launch_move_d<READ, TX, TS, 16>(p, s);
        case 32: return launch_move_d<READ, TX, TS, 32>(p, s);
        case 64: return launch_move_d<READ, TX, TS, 64>(p, s);
        case 128: return launch_move_d<READ, TX, TS, 128>(p, s);
        case 256: return launch_move_d<READ, TX, TS, 256>(p, s);
    }
    return hipErrorInvalidValue;
}

template <bool READ> hipError_t launch_move(const MoveParams &p, int dtype, int store, hipStream_t s) {
    if (dtype == ST_F16 && store == ST_F16) return launch_move_t<READ, f16, f16>(p, s);
    if (dtype == ST_F32 && store == ST_F32) return launch_move_t<READ, float, float>(p, s);
    if (dtype == ST_F16 && store == ST_E4M3) return launch_move_t<READ, f16, e4m3>(p, s);
    if (dtype == ST_F32 && store == ST_E4M3) return launch_move_t<READ, float, e4m3>(p, s);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_append(const MoveParams &p, int dtype, int store, hipStream_t s) { return launch_move<false>(p, dtype, store, s); }
hipError_t launch_read(const MoveParams &p, int dtype, int store, hipStream_t s) { return launch_move<true>(p, dtype, store, s); }

}  // namespace fpa
