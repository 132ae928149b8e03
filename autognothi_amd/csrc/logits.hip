// logits.hip — operators over wide rows of logits (a vocabulary, a large class set): log-probabilities of given tokens with entropy,
// normaliser and the top alternatives; distillation from a teacher's top log-probabilities; the gradients of both.
//
// With x = z / temperature, m a reference of the row and s = sum_i exp(x_i - m):
//     log p_i = (x_i - m) - ln s,   lse = m + ln s,   H = ln s - (1/s) sum_i exp(x_i - m) (x_i - m).
// Everything below is one pass (or few) over the row with (m, s, ...) in fp32; one workgroup per row, no atomics in sums: results are
// bit-reproducible.
#include "common.h"

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_WAVES = LG_THREADS / 64;
constexpr float LG_NEG = -3.402823466e38f;   // the reference of a row (or part of one) that holds nothing above -inf

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int w = 1; w < LG_WAVES; ++w) r += red[w];
    return r;
}
__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int w = 1; w < LG_WAVES; ++w) r = fmaxf(r, red[w]);
    return r;
}
__device__ __forceinline__ unsigned long long block_max_u64(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor(v, o, 64);
        v = u > v ? u : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long r = red[0];
#pragma unroll
    for (int w = 1; w < LG_WAVES; ++w) r = red[w] > r ? red[w] : r;
    return r;
}

// a total order on the logits of a row: by value (-0 = +0, NaN above everything, as torch.topk orders them), ties by the lower index
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float x, int i) {
    return ((unsigned long long)order_key(x) << 32) | (0xFFFFFFFFu - (uint32_t)i);
}

struct RowSums { float m, s, t; };   // reference (in logits), sum of exp, sum of exp * (x - m)

// d = z - m is exact enough at any magnitude (both near the type's lowest value included); a NaN or +inf in the row makes s NaN
template <typename T, bool SKIP>
__device__ RowSums row_sums(const T* __restrict__ z, int V, float inv_t, const uint32_t* skip, float* red) {
    float m = LG_NEG;
    for (int i = threadIdx.x; i < V; i += LG_THREADS)
        if (!SKIP || !((skip[i >> 5] >> (i & 31)) & 1u)) m = fmaxf(m, Store<T>::load(z + i));
    m = block_max(m, red);
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < V; i += LG_THREADS) {
        if (SKIP && ((skip[i >> 5] >> (i & 31)) & 1u)) continue;
        const float x = Store<T>::load(z + i);
        const float d = (x - m) * inv_t;
        const float e = x == -INFINITY ? 0.f : expf(d);
        s += e;
        t += e == 0.f ? 0.f : e * d;
    }
    RowSums r;
    r.m = m;
    r.s = block_sum(s, red);
    r.t = block_sum(t, red);
    return r;
}

template <typename T>
__global__ __launch_bounds__(LG_THREADS) void token_logprobs_kernel(const T* __restrict__ z, int64_t ld, int V, float inv_t,
                                                                    const int64_t* __restrict__ tokens, int top_k, float* __restrict__ logp,
                                                                    float* __restrict__ entropy, float* __restrict__ lse,
                                                                    float* __restrict__ stats, int64_t* __restrict__ top_ids,
                                                                    float* __restrict__ top_logp) {
    __shared__ float red[LG_WAVES];
    __shared__ unsigned long long red64[LG_WAVES];
    const int64_t row = blockIdx.x;
    const T* zr = z + row * ld;
    const RowSums r = row_sums<T, false>(zr, V, inv_t, nullptr, red);
    const bool empty = r.s == 0.f;
    const float log_s = empty ? -INFINITY : logf(r.s);
    if (threadIdx.x == 0) {
        stats[row * 2] = r.m;
        stats[row * 2 + 1] = r.s;
        lse[row] = empty ? -INFINITY : r.m * inv_t + log_s;
        entropy[row] = empty ? 0.f : log_s - r.t / r.s;
        if (tokens) {
            const int64_t t = tokens[row];
            float v = 0.f;
            if (t >= V) v = NAN;
            else if (t >= 0) v = empty ? -INFINITY : (Store<T>::load(zr + t) - r.m) * inv_t - log_s;
            logp[row] = v;
        }
    }
    unsigned long long below = ~0ull;   // (no element has this key: its index would be beyond every row)
    for (int k = 0; k < top_k; ++k) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < V; i += LG_THREADS) {
            const unsigned long long key = order_key(Store<T>::load(zr + i), i);
            if (key < below && key > best) best = key;
        }
        below = block_max_u64(best, red64);
        if (threadIdx.x == 0) {
            const int i = (int)(0xFFFFFFFFu - (uint32_t)below);
            top_ids[row * top_k + k] = i;
            top_logp[row * top_k + k] = empty ? -INFINITY : (Store<T>::load(zr + i) - r.m) * inv_t - log_s;
        }
    }
}

// dz_i = inv_t [ p_i (A + B log p_i) + g_t 1[i = t] + sum_j g_j 1[i = id_j] ],  A = g_lse - g_t - sum_j g_j - g_H H,  B = -g_H
template <typename T>
__global__ __launch_bounds__(LG_THREADS) void token_logprobs_bwd_kernel(const T* __restrict__ z, int64_t ld, int V, float inv_t,
                                                                        const float* __restrict__ stats, const float* __restrict__ entropy,
                                                                        const int64_t* __restrict__ tokens, const float* __restrict__ g_logp,
                                                                        const float* __restrict__ g_entropy, const float* __restrict__ g_lse,
                                                                        int top_k, const int64_t* __restrict__ top_ids,
                                                                        const float* __restrict__ g_top, T* __restrict__ dz, int64_t ldd) {
    __shared__ float red[LG_WAVES];
    const int64_t row = blockIdx.x;
    const T* zr = z + row * ld;
    T* dr = dz + row * ldd;
    const float m = stats[row * 2], s = stats[row * 2 + 1];
    if (s == 0.f) {   // nothing in the row has a probability
        for (int i = threadIdx.x; i < V; i += LG_THREADS) Store<T>::store(dr + i, 0.f);
        return;
    }
    const float inv_s = 1.f / s, log_s = logf(s);
    const int64_t t = tokens ? tokens[row] : -1;
    const float gt = t < 0 || !g_logp ? 0.f : t < V ? g_logp[row] : NAN;
    const float gh = g_entropy ? g_entropy[row] : 0.f;
    float gs = 0.f;
    if (g_top)
        for (int j = threadIdx.x; j < top_k; j += LG_THREADS) gs += g_top[row * top_k + j];
    const float A = (g_lse ? g_lse[row] : 0.f) - gt - block_sum(gs, red) - gh * entropy[row], B = -gh;
    for (int i = threadIdx.x; i < V; i += LG_THREADS) {
        const float d = (Store<T>::load(zr + i) - m) * inv_t;
        const float p = expf(d) * inv_s;
        Store<T>::store(dr + i, p == 0.f ? 0.f : inv_t * p * (A + B * (d - log_s)));
    }
    __syncthreads();
    // the listed places again, with what lands on them alone (top ids are distinct; the given token may be one of them)
    for (int j = threadIdx.x; j <= top_k; j += LG_THREADS) {
        const bool is_token = j == top_k;
        if (is_token ? (t < 0 || t >= V) : !g_top) continue;
        const int64_t i = is_token ? t : top_ids[row * top_k + j];
        if (i < 0 || i >= V) continue;
        float g = is_token ? gt : g_top[row * top_k + j];
        if (!is_token && i == t) g += gt;
        bool dup = false;
        if (is_token && g_top)
            for (int q = 0; q < top_k; ++q) dup |= top_ids[row * top_k + q] == i;
        if (dup) continue;
        const float d = (Store<T>::load(zr + i) - m) * inv_t;
        const float p = expf(d) * inv_s;
        Store<T>::store(dr + i, inv_t * ((p == 0.f ? 0.f : p * (A + B * (d - log_s))) + g));
    }
}

struct Teacher { float Q, rest, qlogq; };

// the list's masses q_j (LDS) and their sums; ids below 0 are empty slots, ids beyond the row make every sum NaN
__device__ Teacher teacher_row(const int64_t* __restrict__ ids, const void* __restrict__ logp, int logp_dtype, int64_t at, int K, int V, bool tail,
                               int* sid, float* sq, float* red) {
    const int tid = threadIdx.x;
    float lp = -INFINITY;
    int id = -1;
    if (tid < K) {
        const int64_t i = ids[at + tid];
        id = i < 0 ? -1 : i >= V ? V : (int)i;
        lp = logp_dtype == AG_BF16 ? bf16_to_f32(((const bf16_t*)logp)[at + tid]) : ((const float*)logp)[at + tid];
        if (id < 0) lp = -INFINITY;
        if (id == V) lp = NAN;
    }
    const float m = block_max(lp, red);
    if (!tail) {
        const float e = lp == -INFINITY ? 0.f : expf(lp - m);
        const float s = block_sum(e, red);
        lp = s == 0.f ? -INFINITY : (lp - m) - logf(s);
    }
    const float q = lp == -INFINITY ? 0.f : expf(lp);
    if (tid < K) { sid[tid] = id; sq[tid] = q; }
    Teacher r;
    r.Q = block_sum(q, red);
    r.qlogq = block_sum(q == 0.f ? 0.f : q * lp, red);
    // 1 - sum q without the cancellation of its largest term: -expm1(lp) of that one, minus the others
    r.rest = 0.f;
    if (tail) {
        __shared__ int first;
        if (tid == 0) first = K;
        __syncthreads();
        if (tid < K && lp == m) atomicMin(&first, tid);
        __syncthreads();
        const float part = tid == first && lp > -INFINITY ? -expm1f(lp) : -q;
        const float sum = block_sum(part, red);
        r.rest = m == -INFINITY ? 1.f : fmaxf(sum, 0.f);
        if (r.Q != r.Q) r.rest = r.Q;
    }
    return r;
}

// L = tau^2 [ sum_j q_j (ln q_j - ln p_j) + rest (ln rest - ln p_off) ];  dL/dz_i = tau [ p_i (Q + rest) - q_i - 1[i off the list] rest p_i / p_off ]
// stats (m_off, a, m, on): the gradient is tau g a exp((z - m_off) / tau) off the list and tau g (on exp((z - m) / tau) - q) on it
template <typename T, bool TAIL>
__global__ __launch_bounds__(LG_THREADS) void topk_distill_kernel(const T* __restrict__ z, int64_t ld, int V, float tau, float inv_t,
                                                                  const int64_t* __restrict__ ids, const void* __restrict__ t_logp, int t_dtype, int K,
                                                                  const float* __restrict__ weights, float* __restrict__ row_loss,
                                                                  float* __restrict__ stats) {
    extern __shared__ uint32_t bits[];
    __shared__ float red[LG_WAVES];
    __shared__ int sid[LG_THREADS];
    __shared__ float sq[LG_THREADS];
    __shared__ int distinct;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const T* zr = z + row * ld;
    if (weights && weights[row] == 0.f) {
        if (tid == 0) row_loss[row] = 0.f;
        if (tid < 4) stats[row * 4 + tid] = 0.f;
        return;
    }
    Teacher tc = teacher_row(ids, t_logp, t_dtype, row * K, K, V, TAIL, sid, sq, red);
    if (TAIL) {
        if (tid == 0) distinct = 0;
        for (int i = tid; i < (V + 31) / 32; i += LG_THREADS) bits[i] = 0u;
        __syncthreads();
        if (tid < K && sid[tid] >= 0 && sid[tid] < V) {
            const uint32_t b = 1u << (sid[tid] & 31);
            if (!(atomicOr(&bits[sid[tid] >> 5], b) & b)) atomicAdd(&distinct, 1);
        }
        __syncthreads();
        if (distinct == V && tc.rest == tc.rest) tc.rest = 0.f;   // no token is off the list
    }
    const RowSums off = row_sums<T, TAIL>(zr, V, inv_t, bits, red);   // over the tokens off the list (TAIL) or over all of them
    const bool mine = tid < K && sid[tid] >= 0 && sid[tid] < V;       // this thread's slot names a token
    bool first = mine;                                                // ... that no earlier slot names
    float x = LG_NEG;
    if (mine) {
        x = Store<T>::load(zr + sid[tid]);
        for (int j = 0; j < tid; ++j) first &= sid[j] != sid[tid];
    }
    float m = off.m, s = off.s;
    if (TAIL) {
        m = fmaxf(m, block_max(x, red));
        s = block_sum(first && x != -INFINITY ? expf((x - m) * inv_t) : 0.f, red) + (off.s == 0.f ? 0.f : off.s * expf((off.m - m) * inv_t));
    }
    const bool empty = s == 0.f;
    const float log_s = empty ? -INFINITY : logf(s);
    const float q = tid < K ? sq[tid] : 0.f;
    const float cross = block_sum(q == 0.f ? 0.f : !mine ? NAN : q * (empty ? INFINITY : log_s - (x - m) * inv_t), red);
    if (tid == 0) {
        float L = tc.qlogq + cross;
        const float log_off = off.s == 0.f ? -INFINITY : (off.m - m) * inv_t + logf(off.s) - log_s;
        if (TAIL && tc.rest != 0.f) L += tc.rest * (logf(tc.rest) - log_off);
        row_loss[row] = tau * tau * L;
        const float on = empty ? 0.f : (tc.Q + tc.rest) / s;
        stats[row * 4] = off.m;
        stats[row * 4 + 1] = !TAIL ? on : off.s == 0.f ? 0.f : on * expf((off.m - m) * inv_t) - tc.rest / off.s;
        stats[row * 4 + 2] = empty ? -INFINITY : m;
        stats[row * 4 + 3] = on;
    }
}

template <typename T>
__global__ __launch_bounds__(LG_THREADS) void topk_distill_bwd_kernel(const T* __restrict__ z, int64_t ld, int V, float tau, float inv_t,
                                                                      const int64_t* __restrict__ ids, const void* __restrict__ t_logp, int t_dtype,
                                                                      int K, const float* __restrict__ weights, float weight0, int tail,
                                                                      const float* __restrict__ stats, const float* __restrict__ g_loss,
                                                                      const float* __restrict__ g_row, T* __restrict__ dz, int64_t ldd) {
    __shared__ float red[LG_WAVES];
    __shared__ int sid[LG_THREADS];
    __shared__ float sq[LG_THREADS];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const T* zr = z + row * ld;
    T* dr = dz + row * ldd;
    const float w = weights ? weights[row] : weight0;
    const float m_off = stats[row * 4], a = stats[row * 4 + 1], m = stats[row * 4 + 2], on = stats[row * 4 + 3];
    if (w == 0.f || m == -INFINITY) {   // the row takes no part, or none of its logits is above -inf
        for (int i = tid; i < V; i += LG_THREADS) Store<T>::store(dr + i, 0.f);
        return;
    }
    const float g = tau * ((g_loss ? w * g_loss[0] : 0.f) + (g_row ? g_row[row] : 0.f) + (!g_loss && !g_row ? w : 0.f));
    teacher_row(ids, t_logp, t_dtype, row * K, K, V, tail != 0, sid, sq, red);
    for (int i = tid; i < V; i += LG_THREADS) {
        const float e = expf((Store<T>::load(zr + i) - m_off) * inv_t);
        Store<T>::store(dr + i, e == 0.f ? 0.f : g * a * e);
    }
    __syncthreads();
    if (tid < K && sid[tid] >= 0 && sid[tid] < V) {
        float q = 0.f;
        bool first = true;
        for (int j = 0; j < K; ++j)
            if (sid[j] == sid[tid]) { q += sq[j]; first &= j >= tid; }
        const float e = expf((Store<T>::load(zr + sid[tid]) - m) * inv_t);
        if (first) Store<T>::store(dr + sid[tid], g * ((e == 0.f ? 0.f : e * on) - q));
    }
}

// sum_n w_n L_n in a fixed order
__global__ __launch_bounds__(1024) void weighted_sum_kernel(const float* __restrict__ row_loss, const float* __restrict__ weights, float weight0, int N,
                                                            float* __restrict__ loss) {
    __shared__ double red[16];
    double acc = 0.0;
    for (int i = threadIdx.x; i < N; i += 1024) {
        const float w = weights ? weights[i] : weight0;
        if (w != 0.f) acc += (double)w * (double)row_loss[i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double r = 0.0;
        for (int w = 0; w < 16; ++w) r += red[w];
        loss[0] = (float)r;
    }
}

int check_rows(const char* who, const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature) {
    AG_REQUIRE(N >= 0 && V >= 1 && V <= AG_LOGITS_MAX_V, "%s: %d rows x %d logits (1 to %d logits per row)", who, N, V, AG_LOGITS_MAX_V);
    AG_REQUIRE(d_logits || N == 0, "%s: null pointer", who);
    AG_REQUIRE(dtype == AG_F32 || dtype == AG_BF16, "%s: dtype %d (AG_F32 or AG_BF16)", who, dtype);
    AG_REQUIRE(ld >= 0, "%s: row stride %lld", who, (long long)ld);
    AG_REQUIRE(temperature > 0.f && temperature <= 3.0e38f, "%s: temperature %g (a positive number)", who, (double)temperature);
    return AG_OK;
}

}  // namespace

extern "C" int ag_token_logprobs(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_tokens, int top_k,
                                 float* d_logp, float* d_entropy, float* d_lse, float* d_stats, int64_t* d_top_ids, float* d_top_logp,
                                 void* stream) {
    if (int rc = check_rows("ag_token_logprobs", d_logits, ld, N, V, dtype, temperature)) return rc;
    AG_REQUIRE(top_k >= 0 && top_k <= AG_LOGITS_MAX_TOP && top_k <= V, "ag_token_logprobs: top_k = %d (0 to min(%d, %d logits))", top_k,
               AG_LOGITS_MAX_TOP, V);
    if (N == 0) return AG_OK;
    AG_REQUIRE(d_entropy && d_lse && d_stats && (!d_tokens || d_logp) && (top_k == 0 || (d_top_ids && d_top_logp)), "ag_token_logprobs: null pointer");
    const float inv_t = (float)(1.0 / (double)temperature);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == AG_BF16)
        hipLaunchKernelGGL(token_logprobs_kernel<bf16_t>, dim3(N), dim3(LG_THREADS), 0, s, (const bf16_t*)d_logits, ld, V, inv_t, d_tokens, top_k, d_logp,
                           d_entropy, d_lse, d_stats, d_top_ids, d_top_logp);
    else
        hipLaunchKernelGGL(token_logprobs_kernel<float>, dim3(N), dim3(LG_THREADS), 0, s, (const float*)d_logits, ld, V, inv_t, d_tokens, top_k, d_logp,
                           d_entropy, d_lse, d_stats, d_top_ids, d_top_logp);
    AG_LAUNCH_CHECK();
    return AG_OK;
}

extern "C" int ag_token_logprobs_bwd(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const float* d_stats,
                                     const float* d_entropy, const int64_t* d_tokens, const float* d_g_logp, const float* d_g_entropy,
                                     const float* d_g_lse, int top_k, const int64_t* d_top_ids, const float* d_g_top_logp, void* d_dlogits,
                                     int64_t ldd, void* stream) {
    if (int rc = check_rows("ag_token_logprobs_bwd", d_logits, ld, N, V, dtype, temperature)) return rc;
    AG_REQUIRE(top_k >= 0 && top_k <= AG_LOGITS_MAX_TOP && top_k <= V, "ag_token_logprobs_bwd: top_k = %d (0 to min(%d, %d logits))", top_k,
               AG_LOGITS_MAX_TOP, V);
    if (N == 0) return AG_OK;
    AG_REQUIRE(d_stats && d_entropy && d_dlogits && (!d_g_logp || d_tokens) && (!d_g_top_logp || d_top_ids), "ag_token_logprobs_bwd: null pointer");
    AG_REQUIRE(ldd >= V, "ag_token_logprobs_bwd: gradient row stride %lld < %d logits", (long long)ldd, V);
    const float inv_t = (float)(1.0 / (double)temperature);
    hipStream_t s = (hipStream_t)stream;
    if (!d_g_top_logp) top_k = 0;
    if (!d_g_logp) d_tokens = nullptr;
    if (dtype == AG_BF16)
        hipLaunchKernelGGL(token_logprobs_bwd_kernel<bf16_t>, dim3(N), dim3(LG_THREADS), 0, s, (const bf16_t*)d_logits, ld, V, inv_t, d_stats, d_entropy,
                           d_tokens, d_g_logp, d_g_entropy, d_g_lse, top_k, d_top_ids, d_g_top_logp, (bf16_t*)d_dlogits, ldd);
    else
        hipLaunchKernelGGL(token_logprobs_bwd_kernel<float>, dim3(N), dim3(LG_THREADS), 0, s, (const float*)d_logits, ld, V, inv_t, d_stats, d_entropy,
                           d_tokens, d_g_logp, d_g_entropy, d_g_lse, top_k, d_top_ids, d_g_top_logp, (float*)d_dlogits, ldd);
    AG_LAUNCH_CHECK();
    return AG_OK;
}

static int check_teacher(const char* who, int V, const void* ids, const void* t_logp, int t_dtype, int K, int N) {
    AG_REQUIRE(K >= 1 && K <= AG_LOGITS_MAX_TOP, "%s: lists of %d tokens (1 to %d)", who, K, AG_LOGITS_MAX_TOP);
    AG_REQUIRE(N == 0 || (ids && t_logp), "%s: null pointer", who);
    AG_REQUIRE(t_dtype == AG_F32 || t_dtype == AG_BF16, "%s: teacher dtype %d (AG_F32 or AG_BF16)", who, t_dtype);
    return AG_OK;
}

template <typename T>
static int distill_bwd(const void* d_logits, int64_t ld, int N, int V, float temperature, const int64_t* d_ids, const void* d_t_logp, int t_dtype, int K,
                       const float* d_weights, int tail, const float* d_stats, const float* d_g_loss, const float* d_g_row, void* d_dlogits,
                       int64_t ldd, hipStream_t s) {
    hipLaunchKernelGGL(topk_distill_bwd_kernel<T>, dim3(N), dim3(LG_THREADS), 0, s, (const T*)d_logits, ld, V, temperature,
                       (float)(1.0 / (double)temperature), d_ids, d_t_logp, t_dtype, K, d_weights, (float)(1.0 / N), tail, d_stats, d_g_loss, d_g_row,
                       (T*)d_dlogits, ldd);
    AG_LAUNCH_CHECK();
    return AG_OK;
}

template <typename T>
static int distill_fwd(const void* d_logits, int64_t ld, int N, int V, float temperature, const int64_t* d_ids, const void* d_t_logp, int t_dtype, int K,
                       const float* d_weights, int tail, float* d_row_loss, float* d_stats, hipStream_t s) {
    const float inv_t = (float)(1.0 / (double)temperature);
    if (tail)
        hipLaunchKernelGGL((topk_distill_kernel<T, true>), dim3(N), dim3(LG_THREADS), (size_t)((V + 31) / 32) * 4, s, (const T*)d_logits, ld, V, temperature,
                           inv_t, d_ids, d_t_logp, t_dtype, K, d_weights, d_row_loss, d_stats);
    else
        hipLaunchKernelGGL((topk_distill_kernel<T, false>), dim3(N), dim3(LG_THREADS), 0, s, (const T*)d_logits, ld, V, temperature, inv_t, d_ids, d_t_logp,
                           t_dtype, K, d_weights, d_row_loss, d_stats);
    AG_LAUNCH_CHECK();
    return AG_OK;
}

extern "C" int ag_topk_distill(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_teacher_ids,
                               const void* d_teacher_logp, int teacher_dtype, int K, const float* d_weights, int tail, float* d_row_loss,
                               float* d_loss, float* d_stats, void* d_dlogits, int64_t ldd, void* stream) {
    if (int rc = check_rows("ag_topk_distill", d_logits, ld, N, V, dtype, temperature)) return rc;
    if (int rc = check_teacher("ag_topk_distill", V, d_teacher_ids, d_teacher_logp, teacher_dtype, K, N)) return rc;
    AG_REQUIRE(N >= 1 && d_row_loss && d_loss && d_stats, "ag_topk_distill: no rows or a null pointer");
    AG_REQUIRE(!d_dlogits || ldd >= V, "ag_topk_distill: gradient row stride %lld < %d logits", (long long)ldd, V);
    hipStream_t s = (hipStream_t)stream;
    int rc = dtype == AG_BF16 ? distill_fwd<bf16_t>(d_logits, ld, N, V, temperature, d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, tail,
                                                    d_row_loss, d_stats, s)
                              : distill_fwd<float>(d_logits, ld, N, V, temperature, d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, tail,
                                                   d_row_loss, d_stats, s);
    if (rc) return rc;
    hipLaunchKernelGGL(weighted_sum_kernel, dim3(1), dim3(1024), 0, s, d_row_loss, d_weights, (float)(1.0 / N), N, d_loss);
    AG_LAUNCH_CHECK();
    if (!d_dlogits) return AG_OK;
    return ag_topk_distill_bwd(d_logits, ld, N, V, dtype, temperature, d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, tail, d_stats, nullptr,
                               nullptr, d_dlogits, ldd, stream);
}

extern "C" int ag_topk_distill_bwd(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_teacher_ids,
                                   const void* d_teacher_logp, int teacher_dtype, int K, const float* d_weights, int tail, const float* d_stats,
                                   const float* d_g_loss, const float* d_g_row_loss, void* d_dlogits, int64_t ldd, void* stream) {
    if (int rc = check_rows("ag_topk_distill_bwd", d_logits, ld, N, V, dtype, temperature)) return rc;
    if (int rc = check_teacher("ag_topk_distill_bwd", V, d_teacher_ids, d_teacher_logp, teacher_dtype, K, N)) return rc;
    AG_REQUIRE(N >= 1 && d_stats && d_dlogits, "ag_topk_distill_bwd: no rows or a null pointer");
    AG_REQUIRE(ldd >= V, "ag_topk_distill_bwd: gradient row stride %lld < %d logits", (long long)ldd, V);
    hipStream_t s = (hipStream_t)stream;
    return dtype == AG_BF16 ? distill_bwd<bf16_t>(d_logits, ld, N, V, temperature, d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, tail, d_stats,
                                                  d_g_loss, d_g_row_loss, d_dlogits, ldd, s)
                            : distill_bwd<float>(d_logits, ld, N, V, temperature, d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, tail, d_stats,
                                                 d_g_loss, d_g_row_loss, d_dlogits, ldd, s);
}
