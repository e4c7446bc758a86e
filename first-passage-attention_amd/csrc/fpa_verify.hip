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
#include "fpa_common.h"
#include "fpa_serve.h"

namespace fpa {

namespace {

constexpr int VT = 1024, VW = VT / 64;

template <typename T> __device__ __forceinline__ double prob(const T *row, int64_t v) { return (double)(float)row[v]; }

__device__ __forceinline__ bool positive(double x) {  // > 0 and finite
    return x > 0.0 && x <= 1.7976931348623157e308;
}

// Weight of token v: p, or what it has more than q.
template <typename T, bool Q> __device__ __forceinline__ double weight(const T *p, const T *q, int64_t x, int64_t v) {
    double w = prob(p, v);
    if constexpr (Q) {
        if (q)
            w -= prob(q, v);
        else if (v == x)
            w = 0.0;
    }
    return w < 0.0 ? 0.0 : w;  // NaN stays: the row has no sum then
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// The lowest v with sum_{v' <= v} w > r * sum w; -1 when the weights have no positive finite sum.
template <typename T, bool Q>
__device__ int64_t draw(const T *p, const T *q, int64_t x, int V, double r, double *seg, int *found) {
    const int lane = thread_x() % 64, wave = thread_x() / 64;
    const int per = (V + VW - 1) / VW, v0 = min(wave * per, V), v1 = min(v0 + per, V);
    double s = 0.0;
    for (int v = v0 + lane; v < v1; v += 64) s += weight<T, Q>(p, q, x, v);
    s = wave_sum(s);
    __syncthreads();  // seg and found are free
    if (lane == 0) seg[wave] = s;
    if (thread_x() == 0) *found = -1;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < VW; ++w) total += seg[w];
    if (!positive(total)) return -1;
    // the first segment whose end passes the target, or the last with any weight
    const double target = r * total;
    double before = 0.0, at = 0.0;
    int pick = -1, lastw = 0;
    for (int w = 0; w < VW; ++w) {
        if (seg[w] > 0.0) lastw = w;
        if (pick < 0 && before + seg[w] > target) {
            pick = w;
            at = before;
        }
        before += seg[w];
    }
    if (pick < 0) {
        pick = lastw;
        at = before - seg[lastw];
    }
    if (wave == pick) {
        int64_t token = -1, least = -1;  // least: the last token with weight, for sums that round below the target
        for (int v = v0; v < v1 && token < 0; v += 64) {
            const double w = v + lane < v1 ? weight<T, Q>(p, q, x, v + lane) : 0.0;
            double c = w;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double u = __shfl_up(c, o, 64);
                if (lane >= o) c += u;
            }
            const uint64_t some = __ballot(w > 0.0), over = __ballot(w > 0.0 && at + c > target);
            if (over) token = v + __builtin_ctzll(over);
            if (some) least = v + 63 - __builtin_clzll(some);
            at += __shfl(c, 63, 64);
        }
        if (lane == 0) *found = (int)(token >= 0 ? token : least);
    }
    __syncthreads();
    return *found;
}

template <typename T> __global__ __launch_bounds__(VT) void fpa_verify_kernel(VerifyParams a) {
    __shared__ double seg[VW];
    __shared__ int found, first, none;
    const int b = group_x(), lane = thread_x() % 64;
    const T *p = static_cast<const T *>(a.target) + (int64_t)b * a.stb;
    const T *q = a.draft ? static_cast<const T *>(a.draft) + (int64_t)b * a.sdb : nullptr;
    const int64_t *x = a.tokens + (int64_t)b * a.sxb;
    const float *u = a.accept_u + (int64_t)b * a.sub;
    if (thread_x() < 64) {  // the first draft that is not accepted, and whether there is a token there at all
        int n = a.N, end = 1;
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
                n = i0 + k;
                end = (there >> k & 1) == 0;
                break;
            }
        }
        if (lane == 0) {
            first = n;
            none = end;
        }
    }
    __syncthreads();
    const int n = first;
    const T *pr = p + (int64_t)n * a.stn;
    const double r = (double)a.sample_u[b];
    int64_t token = -1;
    if (!none) token = draw<T, true>(pr, q ? q + (int64_t)n * a.sdn : nullptr, x[n], a.V, r, seg, &found);
    if (token < 0) token = draw<T, false>(pr, nullptr, -1, a.V, r, seg, &found);
    for (int i = thread_x(); i <= a.N; i += VT) a.out[(int64_t)b * (a.N + 1) + i] = i < n ? x[i] : i == n ? token : -1;
    if (thread_x() == 0) a.accepted[b] = n;
}

}  // namespace

hipError_t launch_verify(const VerifyParams &p, int dtype, hipStream_t s) {
    if (dtype == ST_F16)
        hipLaunchKernelGGL((fpa_verify_kernel<f16>), dim3(p.B), dim3(VT), 0, s, p);
    else
        hipLaunchKernelGGL((fpa_verify_kernel<float>), dim3(p.B), dim3(VT), 0, s, p);
    return hipGetLastError();
}

}  // namespace fpa
