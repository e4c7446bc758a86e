// fpa_verify.hip -- accepting or rejecting drafted tokens against the target model's probabilities.
//
// Token x_i of a sequence, drawn from the draft's q_i, is accepted with probability min(1, p_i(x_i) / q_i(x_i)): with
// the given uniform u_i in [0, 1), while u_i q_i(x_i) < p_i(x_i).  At the first rejection j the next token is
// drawn from max(p_j - q_j, 0), normalised, which makes the outcome distributed as p_j; when all are accepted, from
// the target's row behind the last.  Drafts without probabilities count as certain (q = 1 at x_i, else 0).
//
// Every number is a probability in fp32 or fp16 and everything computed from them is fp64: u q is exact (two 24-bit
// factors), p - q all but exact, and the running sum over the vocabulary is what the drawn token is decided by,
// so its rounding (2^-53 a term) has to lie far below the gaps between tokens; in fp32 another order of summation
// would draw another token now and then.
//
// Bound by a chain: the gathers of the drafted tokens' probabilities, two rows of the vocabulary a sequence read once (65 MB at B64
// V128003 fp32), and the draw within a quarter of a span by each sequence's last workgroup: 29 us there, of which the rows take
// about 15 (4.4 TB/s) and the draw 8 to 10; one sequence of V32000 8 us.  One workgroup a sequence took 177.
#include "fpa_common.h"
#include "fpa_serve.h"

namespace fpa {

namespace {

constexpr int VT = 256, VW = VT / 64;

template <typename T> __device__ __forceinline__ double prob(const T *row, int64_t v) { return (double)(float)row[v]; }

__device__ __forceinline__ bool positive(double x) {  // > 0 and finite
    return x > 0.0 && x <= 1.7976931348623157e308;
}
__device__ __forceinline__ double above(double w) { return w < 0.0 ? 0.0 : w; }  // NaN stays: the row has no sum then

// What is drawn from: row n of the target, less the draft's row unless `whole`.
template <typename T> struct Row {
    const T *p, *q;
    int64_t x;  // the drafted token, which has weight 0 where the drafts have no probabilities
    __device__ __forceinline__ double target(int64_t v) const { return above(prob(p, v)); }
    __device__ __forceinline__ double rest(int64_t v) const {  // what the target has more than the draft
        if (q) return above(prob(p, v) - prob(q, v));
        return v == x ? 0.0 : above(prob(p, v));
    }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// The first draft that is not accepted (N: none), by one wave; `none`: there is no token there.
template <typename T> __device__ int first_rejected(const VerifyParams &a, const T *p, const T *q, const int64_t *x, const float *u, bool &none) {
    const int lane = thread_x() % 64;
    none = true;
    for (int i0 = 0; i0 < a.N; i0 += 64) {
        const int i = i0 + lane;
        bool in = false, ok = false;
        if (i < a.N) {
            const int64_t t = x[i];
            in = t >= 0 && t < a.V;
            if (in) {
                const double qx = q ? prob(q + (int64_t)i * a.sdn, t) : 1.0;
                ok = (double)u[i] * qx < prob(p + (int64_t)i * a.stn, t);
            }
        }
        const uint64_t stop = __ballot(i < a.N && !ok), there = __ballot(in);
        if (stop) {
            const int k = __builtin_ctzll(stop);
            none = (there >> k & 1) == 0;
            return i0 + k;
        }
    }
    return a.N;
}

// Inclusive sums of one value per thread in thread order; total gets the sum of all.
__device__ __forceinline__ double block_sums(double x, double *part, double &total) {
    const int lane = thread_x() % 64, wave = thread_x() / 64;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(x, o, 64);
        if (lane >= o) x += u;
    }
    __syncthreads();  // part is free
    if (lane == 63) part[wave] = x;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < VW; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + x;
}
// The lowest thread for which `over` holds, else the highest for which `some` holds, else -1.
__device__ __forceinline__ int block_pick(bool over, bool some, int *pick) {
    __syncthreads();
    if (thread_x() == 0) {
        pick[0] = VT;
        pick[1] = -1;
    }
    __syncthreads();
    const uint64_t o = __ballot(over), s = __ballot(some);
    if (thread_x() % 64 == 0) {
        const int t0 = thread_x();
        if (o) atomicMin(&pick[0], t0 + __builtin_ctzll(o));
        if (s) atomicMax(&pick[1], t0 + 63 - __builtin_clzll(s));
    }
    __syncthreads();
    return pick[0] < VT ? pick[0] : pick[1];
}

// Values that another workgroup of this launch reads: agent-scope accesses, past the caches that the XCDs do not share.
__device__ __forceinline__ void put(double *p, double x) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get(const double *p) {
    return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// One workgroup a span of a sequence's row; each finds the rejected position for itself, and each wave sums a quarter of the
// span: sums[b][VW * span + wave] = (rest, target).  The workgroup that finishes a sequence's last span draws the token:
// the quarter that the target falls into, then the token in it; sums that round below the target fall to the last token with
// any weight.
template <typename T> __global__ __launch_bounds__(VT) void fpa_verify_kernel(VerifyParams a) {
    __shared__ double part[VW], at;
    __shared__ int first, none, last, pick[2], found;
    const int b = group_y(), span = group_x(), tid = thread_x(), lane = tid % 64, wave = tid / 64;
    const T *p = static_cast<const T *>(a.target) + (int64_t)b * a.stb;
    const T *q = a.draft ? static_cast<const T *>(a.draft) + (int64_t)b * a.sdb : nullptr;
    const int64_t *x = a.tokens + (int64_t)b * a.sxb;
    if (wave == 0) {
        bool no;
        const int n = first_rejected(a, p, q, x, a.accept_u + (int64_t)b * a.sub, no);
        if (lane == 0) {
            first = n;
            none = no;
        }
    }
    __syncthreads();
    const int n = first;
    const bool no = none;
    const Row<T> row = {p + (int64_t)n * a.stn, q && !no ? q + (int64_t)n * a.sdn : nullptr, no ? -1 : x[n]};
    const int quarter = a.span / VW, subs = a.spans * VW;
    double *sums = a.sums + 2 * (int64_t)b * subs;
    {
        const int v0 = (int)min((int64_t)span * a.span + wave * quarter, (int64_t)a.V), v1 = min(v0 + quarter, a.V);
        double rest = 0.0, target = 0.0;
#pragma unroll 8
        for (int v = v0 + lane; v < v1; v += 64) {
            rest += row.rest(v);
            target += row.target(v);
        }
        rest = wave_sum(rest);
        target = wave_sum(target);
        if (lane == 0) {
            put(sums + 2 * (span * VW + wave), rest);
            put(sums + 2 * (span * VW + wave) + 1, target);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    }
    __syncthreads();
    if (tid == 0) {
        int32_t *count = a.counts + b;
        last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == a.spans;
        if (last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    }
    __syncthreads();
    if (!last) return;

    // a thread's quarters: `each` neighbouring ones
    const int each = (subs + VT - 1) / VT, s0 = min(tid * each, subs), s1 = min(s0 + each, subs);
    double rest = 0.0, target = 0.0;
    for (int s = s0; s < s1; ++s) {
        rest += get(sums + 2 * s);
        target += get(sums + 2 * s + 1);
    }
    double total;
    double upto = block_sums(rest, part, total);
    const bool use_rest = !no && positive(total);
    if (!use_rest) upto = block_sums(target, part, total);
    int64_t token = -1;
    if (positive(total)) {
        const double goal = (double)a.sample_u[b] * total, mine = use_rest ? rest : target;
        int who = block_pick(mine > 0.0 && upto > goal, mine > 0.0, pick);
        if (tid == who) {
            double run = s0 == 0 ? 0.0 : upto - mine, last_run = run;
            int in = s0;
            for (int s = s0; s < s1; ++s) {
                const double w = get(sums + 2 * s + !use_rest);
                if (w > 0.0) {
                    in = s;
                    last_run = run;
                    if (run + w > goal) break;
                }
                run += w;
            }
            found = in;
            at = last_run;
        }
        __syncthreads();
        const int64_t f = (int64_t)(found / VW) * a.span + found % VW * quarter;
        const int v0 = (int)f, v1 = (int)min(f + quarter, (int64_t)a.V);
        const int per = (v1 - v0 + VT - 1) / VT, t0 = min(v0 + tid * per, v1), t1 = min(t0 + per, v1);
        double w = 0.0;
        for (int v = t0; v < t1; ++v) w += use_rest ? row.rest(v) : row.target(v);
        const double base = at;
        double all;
        const double end = base + block_sums(w, part, all);
        who = block_pick(w > 0.0 && end > goal, w > 0.0, pick);
        if (tid == who) {
            double run = end - w;
            int in = -1;
            for (int v = t0; v < t1; ++v) {
                const double y = use_rest ? row.rest(v) : row.target(v);
                run += y;
                if (y > 0.0) {
                    in = v;
                    if (run > goal) break;
                }
            }
            found = in;
        }
        __syncthreads();
        token = found;
    }
    for (int i = tid; i <= a.N; i += VT) a.out[(int64_t)b * (a.N + 1) + i] = i < n ? x[i] : i == n ? token : -1;
    if (tid == 0) a.accepted[b] = n;
}

}  // namespace

int verify_span(int64_t B, int64_t V) {
    // Spans of a multiple of 1024 tokens, about 2048 workgroups in all (eight on a CU, 4096 tokens each at the most
    // common sizes).
    int64_t per = (B * V + 2047) / 2048;
    per = per < V ? per : V;
    per = (per + 1023) / 1024 * 1024;
    return (int)per;
}

hipError_t launch_verify(const VerifyParams &p, int dtype, hipStream_t s) {
    if (dtype == ST_F16)
        hipLaunchKernelGGL((fpa_verify_kernel<f16>), dim3(p.spans, p.B), dim3(VT), 0, s, p);
    else
        hipLaunchKernelGGL((fpa_verify_kernel<float>), dim3(p.spans, p.B), dim3(VT), 0, s, p);
    return hipGetLastError();
}

}  // namespace fpa
