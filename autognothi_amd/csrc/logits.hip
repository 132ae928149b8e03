// logits.hip — operators over wide rows of logits (a vocabulary, a large class set): log-probabilities of given tokens with entropy,
// normaliser and the top alternatives; distillation from a teacher's top log-probabilities; the gradients of both.
//
// With x = z / temperature, m a reference of the row and s = sum_i exp(x_i - m):
//     log p_i = (x_i - m) - ln s,   lse = m + ln s,   H = ln s - (1/s) sum_i exp(x_i - m) (x_i - m).
// One pass over the row computes all of it: every lane keeps its own (m, s, t) and moves its reference only when a logit passes it by more
// than LG_SLACK, the lanes are joined once at the end.  A row belongs to a TEAM of 16 or 64 lanes or to a workgroup of 256, 512
// or 1024 threads (a few long ones to several workgroups), and is read in 16-byte pieces ("chunks") from the 16-byte boundary at or below its start, so that
// every whole chunk is one aligned load whatever the row stride is.  Sums are fp32 in a fixed order, no atomics: results are
// bit-reproducible.
#include "common.h"
#include <algorithm>

namespace {

constexpr float LG_NEG = -3.402823466e38f;   // the reference of a row (or part of one) that holds nothing above -inf
// how far (in powers of two) a logit may lie above its lane's reference before the reference moves: 3 keeps |y| <= 3 where the exponentials
// are large, i.e. the rounding of y adds at most 2^-23 ln 2 to a term, and after a few chunks a row no longer moves any reference
constexpr float LG_SLACK = 3.0f;
constexpr float LG_LN2 = 0.69314718055994530942f;

typedef __attribute__((ext_vector_type(4))) uint32_t chunk_t;   // 16 bytes of a row

template <typename T> struct Chunk;   // as E logits
template <> struct Chunk<float> {
    using Bits = uint32_t;
    static constexpr int E = 4;
    static __device__ __forceinline__ void unpack(const chunk_t& r, float (&x)[4]) {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ float pick(const chunk_t& r, int e) {   // (selections, not an array in memory)
        uint32_t a = r.x, b = r.y, c = r.z, d = r.w;
        asm("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
        const uint32_t p = e & 1 ? b : a, q = e & 1 ? d : c;
        return __uint_as_float(e & 2 ? q : p);
    }
    static __device__ __forceinline__ chunk_t pack(const float (&x)[4]) {
        return chunk_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    }
};
template <> struct Chunk<bf16_t> {
    using Bits = bf16_t;
    static constexpr int E = 8;
    static __device__ __forceinline__ void unpack(const chunk_t& r, float (&x)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    }
    static __device__ __forceinline__ float pick(const chunk_t& r, int e) {
        uint32_t a = r.x, b = r.y, c = r.z, d = r.w;
        asm("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
        const uint32_t p = e & 2 ? b : a, q = e & 2 ? d : c, w = e & 4 ? q : p;
        return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
    }
    static __device__ __forceinline__ chunk_t pack(const float (&x)[8]) {
        return chunk_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    }
};

// A row as chunks: chunk c holds the logits [c E - sh, c E - sh + E); those in [first, end) lie inside the row and are aligned 16-byte
// loads.  The up to E - 1 logits before the first and behind the last of them are the row's ends, one for each of 2 E lanes.  Nothing outside
// the row is ever touched.
template <typename T>
struct Row {
    static constexpr int E = Chunk<T>::E;
    const T* z;
    int V, sh, first, end;
    __device__ __forceinline__ Row(const T* p, int v) : z(p), V(v) {
        sh = (int)(((uintptr_t)p & 15) / sizeof(T));
        first = sh ? 1 : 0;
        end = max((v + sh) / E, first);
    }
    __device__ __forceinline__ int full() const { return end - first; }
    __device__ __forceinline__ chunk_t load(int c) const { return *reinterpret_cast<const chunk_t*>(z + (c * E - sh)); }
    __device__ __forceinline__ chunk_t load_past(int c) const { return __builtin_nontemporal_load(reinterpret_cast<const chunk_t*>(z + (c * E - sh))); }
    // one logit's bits, to be made a number (`value`) where it is wanted: nothing waits for the load here
    __device__ __forceinline__ uint32_t bits(int i) const { return reinterpret_cast<const typename Chunk<T>::Bits*>(z)[i]; }
    static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(E == 8 ? b << 16 : b); }
    // the logit at the row's ends that belongs to lane l of the row's threads (-1: none)
    __device__ __forceinline__ int end_index(int l) const {
        if (l < E) return sh && l < min(E - sh, V) ? l : -1;
        const int i = max(end * E - sh, 0) + (l - E);
        return l < 2 * E && i < V ? i : -1;
    }
    // the chunk's place in another row of the same length (at the logits' alignment: the hardware takes any)
    __device__ __forceinline__ void store(T* d, int c, const float (&x)[E]) const { store<false>(d, c, x); }
    template <bool PAST> __device__ __forceinline__ void store(T* d, int c, const float (&x)[E]) const {
        typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t any_chunk_t;
        any_chunk_t* to = reinterpret_cast<any_chunk_t*>(d + (c * E - sh));
        const any_chunk_t v = Chunk<T>::pack(x);
        if (PAST) __builtin_nontemporal_store(v, to);
        else *to = v;
    }
};

// ---- joining lanes: the value of every lane of a team of W <= 64 lanes, the same bits on all of them ---------------------------
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int W, typename F> __device__ __forceinline__ float lanes_join(float v, F f) {
    static_assert(W == 4 || W == 8 || W == 16 || W == 64, "team of lanes");
    v = f(v, dpp<0xB1>(v));                   // quad_perm 1 0 3 2
    v = f(v, dpp<0x4E>(v));                   // quad_perm 2 3 0 1
    if (W >= 8) v = f(v, dpp<0x141>(v));      // row_half_mirror (a quad already agrees)
    if (W >= 16) v = f(v, dpp<0x140>(v));     // row_mirror
    if (W == 64) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
        const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
    }
    return v;
}
// one number that all lanes of a wave want, through the scalar cache (a vector load would queue behind every load of the row in flight)
__device__ __forceinline__ float scalar_load(const float* p) {
    typedef __attribute__((address_space(4))) const float constant_float;
    return *(constant_float*)(uintptr_t)p;
}

struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };

// TH threads that own a row; red: TH / 64 floats of LDS per use (three planes for Acc), only for TH > 64
template <int TH>
struct Team {
    static constexpr int LANES = TH < 64 ? TH : 64, WAVES = TH / 64;
    static __device__ __forceinline__ int rank() { return TH >= 64 && TH < 256 ? threadIdx.x & 63 : threadIdx.x & (TH - 1); }
    // which team of the workgroup this is (one number for the whole wave where a team is a wave: the row's own numbers are scalars then)
    static __device__ __forceinline__ int index() { return TH >= 256 ? 0 : TH == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / TH; }
    static __device__ __forceinline__ void sync() {
        if (TH > 64) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the LDS and the loads / stores of one wave keep their order
    }
    template <typename F> static __device__ __forceinline__ float join(float v, F f, float* red) {
        v = lanes_join<LANES>(v, f);
        if (TH <= 64) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return lanes_join<(WAVES > 1 ? WAVES : 4)>(red[threadIdx.x & (WAVES - 1)], f);
    }
    static __device__ __forceinline__ float sum(float v, float* red) { return join(v, Add(), red); }
    static __device__ __forceinline__ float max(float v, float* red) { return join(v, Max(), red); }
};

struct Acc { float m, s, t; };   // reference (a logit), sum of exp2(y), sum of exp2(y) y,  y = (z - m) c,  c = log2(e) / temperature

// the same sums with respect to the reference `to` >= m (or equal); an empty one stays empty, a NaN a NaN
__device__ __forceinline__ Acc rebase(const Acc& a, float to, float c) {
    const float dm = (a.m - to) * c, f = __builtin_amdgcn_exp2f(dm);
    Acc r;
    r.m = to;
    r.s = a.m == to ? a.s : a.s * f;
    r.t = a.m == to ? a.t : f == 0.f ? a.s * f : f * fmaf(a.s, dm, a.t);
    return r;
}
template <int W> __device__ __forceinline__ Acc lanes_join(const Acc& a, float c) {
    Acc r = rebase(a, lanes_join<W>(a.m, Max()), c);
    r.s = lanes_join<W>(r.s, Add());
    r.t = lanes_join<W>(r.t, Add());
    return r;
}
template <int TH> __device__ __forceinline__ Acc team_join(Acc a, float c, float* red) {
    constexpr int WAVES = TH / 64;
    a = lanes_join<Team<TH>::LANES>(a, c);
    if (TH <= 64) return a;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        float* p = red + 3 * (threadIdx.x >> 6);
        p[0] = a.m; p[1] = a.s; p[2] = a.t;
    }
    __syncthreads();
    const float* p = red + 3 * (threadIdx.x & (WAVES - 1));
    const Acc b = {p[0], p[1], p[2]};
    return lanes_join<(WAVES > 1 ? WAVES : 4)>(b, c);
}

// y = z c - m c in one instruction: the product m c is rounded, so every y of the reference is off by the same `delta`, which is known exactly
// (and taken out of the sums at the end); past 2^20 delta is no longer small and y is computed as (z - m) c.
struct Ref {
    float m, nr, delta;
    bool far;
    __device__ __forceinline__ Ref() : m(LG_NEG), nr(0.f), delta(0.f), far(true) {}   // of nothing yet
    __device__ __forceinline__ Ref(float m_, float c) : m(m_) {
        nr = -(m * c);
        far = !(fabsf(nr) < 1048576.f);
        delta = far ? 0.f : fmaf(m, c, nr);
    }
    __device__ __forceinline__ float y(float x, float c) const { return far ? (x - m) * c : fmaf(x, c, nr); }   // (z - m) c + delta
};

// One lane's running sums.  A chunk costs about 8.5 instruction slots per logit (an exp2 is four of them): unpack, max (two logits an
// instruction), y, exp2, + and the entropy's fma.
template <typename T, bool ENTROPY>
struct Sums {
    static constexpr int E = Chunk<T>::E;
    float c, slack, s = 0.f, t = 0.f;
    float lim = LG_NEG;   // what a logit must pass to move the reference
    float zero;           // 0, or NaN where the reference is `far`: every chunk then takes the guarded form below
    Ref ref;
    __device__ __forceinline__ Sums(float c_) : c(c_), slack(LG_SLACK / c_) { zero = NAN; }
    // (s, t) without the reference's delta
    __device__ __forceinline__ Acc acc() const {
        const float f = __builtin_amdgcn_exp2f(-ref.delta);
        return {ref.m, f * s, f * fmaf(-ref.delta, s, t)};
    }
    __device__ __forceinline__ void refer(float to) {
        const Acc a = rebase(acc(), to, c);
        ref = Ref(to, c);
        lim = to + slack;
        zero = ref.far ? NAN : 0.f;
        const float f = __builtin_amdgcn_exp2f(ref.delta);
        s = f * a.s;
        t = f * fmaf(ref.delta, a.s, a.t);
    }
    __device__ __forceinline__ void add_guarded(float x, float& cs, float& ct) const {
        const float y = ref.y(x, c), p = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(y);
        cs += p;
        if (ENTROPY) ct += p == 0.f ? 0.f : p * y;
    }
    __device__ __forceinline__ void add_one(float x) {
        if (x > lim) refer(x);
        add_guarded(x, s, t);
    }
    // x: the chunk's logits (-inf: none), cmax: the largest of them
    __device__ __forceinline__ void add(const float (&x)[E], float cmax) {
        if (cmax > lim) refer(cmax);
        float cs = zero, ct = zero;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = fmaf(x[e], c, ref.nr), p = __builtin_amdgcn_exp2f(y);
            cs += p;
            if (ENTROPY) ct = fmaf(p, y, ct);
        }
        // 0 * -inf (a masked logit), or a far reference: the same sums, every step guarded
        const float bad = ENTROPY ? ct : cs;
        if (bad != bad) {
            cs = 0.f; ct = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) add_guarded(x[e], cs, ct);
        }
        s += cs;
        t += ct;
    }
};
// exp2((z - m) c) as the sums above have it, at any magnitude
__device__ __forceinline__ float exp2_from(float z, float m, float c) {
    return z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((z - m) * c);
}

template <int E> __device__ __forceinline__ float max_of(const float (&x)[E]) {
    float m = fmaxf(fmaxf(x[0], x[1]), x[2]);
#pragma unroll
    for (int e = 3; e + 1 < E; e += 2) m = fmaxf(fmaxf(m, x[e]), x[e + 1]);
    return fmaxf(m, x[E - 1]);
}

// a total order on the logits of a row: by value (-0 = +0, NaN above everything), ties by the lower index
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {   // (at least -inf)
    k = k < 0x007FFFFFu ? 0x007FFFFFu : k;
    return k == 0xFFFFFFFFu ? NAN : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ unsigned long long order_key(float x, int i) {
    return ((unsigned long long)order_key(x) << 32) | (0xFFFFFFFFu - (uint32_t)i);
}

// ---- token_logprobs -------------------------------------------------------------------------------------------------------------
// Top alternatives of a row that a workgroup owns.  Every lane remembers the largest logit of each of its SLOTS (the chunks it reads, in
// rounds of LG_SLOTS).  Each wave finds the j-th largest of its lanes' maxima, j = ceil(k / waves); the least of them over the waves is a
// bound that at least k logits reach, and few others: the chunks of the slots that reach it (about two per alternative asked for) are read
// again, their logits at or above the bound are the candidates, and every candidate's place is the number of candidates that beat it.
// Rows with more candidates than fit and rows with a NaN take a radix selection over the whole row, in five more passes that load single logits.
// The bound counts pieces, so that is not only rows of many equal logits: where the large logits lie next to each other (a descending row, a band of
// admissible tokens in a row of -inf) up to E k of them reach it, and in a row of fewer than k finite pieces everything does.  8192 x 131072 bf16, k 64:
// random 0.42 ms, descending, a band of 200 tokens or all equal 6.4-7.0; 4096 x 30522 fp32 0.10, descending 0.37, a band 0.66; 8192 x 8000 bf16 0.04 / 0.53.
constexpr int LG_SLOTS = 16;

template <int TH> struct TopLds {
    static constexpr int CAP = TH == 64 ? 256 : 1024;
    int list[CAP];          // slots to read again; the radix selection's counters
    unsigned long long cand[CAP];
    uint32_t bound[16];
    int n_list, n_cand;
};

// a key that at least j and (unless logits are equal) hardly more than j of the wave's G 64 values reach, by bisection between the least lane
// maximum (or nothing) and the largest value.  SHIFT: low key bits that carry nothing (16 for bf16)
template <int G, int SHIFT> __device__ __forceinline__ uint32_t wave_bound(const float (&v)[G], int j) {
    float mine = v[0];
#pragma unroll
    for (int g = 1; g < G; ++g) mine = fmaxf(mine, v[g]);
    const float most = lanes_join<64>(mine, Max());
    uint32_t key[G];
#pragma unroll
    for (int g = 0; g < G; ++g) key[g] = order_key(v[g]) >> SHIFT;
    uint32_t lo = j <= 64 ? order_key(-lanes_join<64>(-mine, Max())) >> SHIFT : 0u, hi = (order_key(most) >> SHIFT) + 1u;
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int enough = j + min(j >> 3, 4) + (j > 4);
    while (hi - lo > 1u) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        int n = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) n += __popcll(__ballot(key[g] >= mid));
        if (n >= j) {
            lo = mid;
            if (n <= enough) break;
        } else {
            hi = mid;
        }
    }
    return lo << SHIFT;
}

// exact: the k-th largest key by radix (four digits of 8 bits over the row), then every larger logit and the first of the equal ones
template <typename T, int TH> __device__ void top_radix(const Row<T>& row, int k, TopLds<TH>& lds) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    int left = k;                       // how many of the logits with the digits found so far are still wanted
    for (int d = 24; d >= 0; d -= 8) {
        for (int i = tid; i < 256; i += TH) lds.list[i] = 0;
        Team<TH>::sync();
        for (int i = tid; i < row.V; i += TH) {
            const uint32_t key = order_key(Store<T>::load(row.z + i));
            if (d != 24 && (key >> (d + 8)) != prefix) continue;
            const int digit = (key >> d) & 255;
            const unsigned long long on = __ballot(1);
            const int one = __builtin_amdgcn_readfirstlane(digit);
            if (__all(digit == one)) {                       // (rows of equal logits: one addition for the wave)
                if ((tid & 63) == __ffsll(on) - 1) atomicAdd(&lds.list[one], __popcll(on));
            } else {
                atomicAdd(&lds.list[digit], 1);
            }
        }
        Team<TH>::sync();
        int digit = 255, above = 0;
        for (; digit > 0; --digit) {                         // (every thread, the same broadcast reads)
            const int n = lds.list[digit];
            if (above + n >= left) break;
            above += n;
        }
        left -= above;
        prefix = d == 24 ? (uint32_t)digit : (prefix << 8) | digit;
        Team<TH>::sync();
    }
    // prefix is the k-th largest key; `left` of the logits equal to it belong to the top, the first ones
    if (tid == 0) { lds.n_cand = 0; lds.n_list = 0; }
    Team<TH>::sync();
    for (int i0 = 0; i0 < row.V; i0 += TH) {
        const int i = i0 + tid;
        const uint32_t key = i < row.V ? order_key(Store<T>::load(row.z + i)) : 0u;
        if (i < row.V && key > prefix) lds.cand[atomicAdd(&lds.n_cand, 1)] = ((unsigned long long)key << 32) | (0xFFFFFFFFu - (uint32_t)i);
        const bool eq = i < row.V && key == prefix;
        const unsigned long long m = __ballot(eq);
        const int before = lds.n_list;                       // equal logits of the rounds so far
        if (before >= left) continue;                        // (uniform: all of them are found, only larger ones are still wanted)
        Team<TH>::sync();
        if ((tid & 63) == 0) lds.bound[tid >> 6] = __popcll(m);
        Team<TH>::sync();
        int at = before;
        for (int w = 0; w < (tid >> 6); ++w) at += (int)lds.bound[w];
        int total = before;
        for (int w = 0; w < TH / 64; ++w) total += (int)lds.bound[w];
        at += __popcll(m & ((1ull << (tid & 63)) - 1ull));
        if (eq && at < left) lds.cand[atomicAdd(&lds.n_cand, 1)] = ((unsigned long long)key << 32) | (0xFFFFFFFFu - (uint32_t)i);
        Team<TH>::sync();
        if (tid == 0) lds.n_list = total;
        Team<TH>::sync();
    }
    Team<TH>::sync();
}

// ln p <= 0 and H >= 0 hold for the numbers, not for their roundings: of a row that is sure of one token, s is 1 and a few roundings.  A value on
// the wrong side is 0 (a NaN stays one).
__device__ __forceinline__ float log_prob(float z, float m, float inv_t, float log_s) {
    const float v = (z - m) * inv_t - log_s;
    return v > 0.f ? 0.f : v;
}
__device__ __forceinline__ float entropy_of(const Acc& a, float log_s) {
    const float h = log_s - LG_LN2 * (a.t / a.s);
    return h < 0.f ? 0.f : h;
}

struct TopOut {
    int64_t* ids;
    float* logp;
    int k;
    float m, inv_t, log_s;
    bool empty;
    unsigned long long* keys = nullptr;   // of a part of a row that starts at logit `base`: the keys instead, for the whole row
    int base = 0;
    __device__ __forceinline__ void write(unsigned long long me, int place) const {
        if (place >= k) return;
        if (keys) { keys[place] = me - (unsigned long long)base; return; }   // (the key's low half counts down)
        ids[place] = (int64_t)(0xFFFFFFFFu - (uint32_t)me);
        logp[place] = empty ? -INFINITY : log_prob(key_value((uint32_t)(me >> 32)), m, inv_t, log_s);
    }
};

// the value of lane ^ J
template <int J> __device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);
    else if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);
    else if constexpr (J < 32) return __builtin_amdgcn_ds_swizzle(v, (J << 10) | 0x1F);
    else return __shfl_xor(v, J, 64);
}
template <int J> __device__ __forceinline__ unsigned long long lane_xor(unsigned long long v) {
    return ((unsigned long long)lane_xor<J>((uint32_t)(v >> 32)) << 32) | lane_xor<J>((uint32_t)v);
}
// One wave sorts 64 R different keys in descending order, key 64 i + lane in q[i]: a bitonic network, step (S, J) compares keys J apart in
// runs of S.  64 keys of 32 bits: 21 steps of one exchange, one comparison and one selection.
template <int R, int S, int J, typename K> __device__ __forceinline__ void sort_steps(K (&q)[R]) {
    const int lane = threadIdx.x & 63;
    if constexpr (J >= 64) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i & (J / 64)) continue;
            const K a = q[i], b = q[i | (J / 64)];
            const bool swap = (a < b) == !((i * 64) & S);
            q[i] = swap ? b : a;
            q[i | (J / 64)] = swap ? a : b;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const K other = lane_xor<J>(q[i]);
            const bool down = S < 64 ? !(lane & S) : !((i * 64) & S), larger = !(lane & J) == down;
            q[i] = (other > q[i]) == larger ? other : q[i];
        }
    }
    if constexpr (J > 1) sort_steps<R, S, J / 2>(q);
    else if constexpr (S < 64 * R) sort_steps<R, 2 * S, S>(q);
}

// One wave, candidates [0, n) of LDS with k <= n <= 256, all different -> the first k of them in order.  A bf16 candidate's 16 value and (up
// to 65536 logits) 16 index bits are one 32-bit key.
template <typename T, int R> __device__ __forceinline__ void place_sorted(const unsigned long long* cand, int n, int V, const TopOut& out) {
    const int lane = threadIdx.x & 63;
    unsigned long long c[R];
#pragma unroll
    for (int i = 0; i < R; ++i) c[i] = lane + 64 * i < n ? cand[lane + 64 * i] : (unsigned long long)(uint32_t)(lane + 64 * i);   // (below every candidate)
    if (Chunk<T>::E == 8 && V <= 65536) {
        uint32_t q[R];
#pragma unroll
        for (int i = 0; i < R; ++i) q[i] = ((uint32_t)(c[i] >> 32) & 0xFFFF0000u) | ((uint32_t)c[i] & 0xFFFFu);
        sort_steps<R, 2, 1>(q);
        // (the low key bits that were dropped: 0 of a positive bf16 logit, ones of a negative one and of a NaN's key)
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (lane + 64 * i < out.k) {
                const uint32_t hi = q[i] & 0xFFFF0000u, full = hi & 0x80000000u && hi != 0xFFFF0000u ? hi : hi | 0xFFFFu;
                out.write(((unsigned long long)full << 32) | 0xFFFF0000u | (q[i] & 0xFFFFu), lane + 64 * i);
            }
    } else {
        sort_steps<R, 2, 1>(c);
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (lane + 64 * i < out.k) out.write(c[i], lane + 64 * i);
    }
}
template <typename T> __device__ __forceinline__ void place_wave(const unsigned long long* cand, int n, int V, const TopOut& out) {
    if (n <= 64) place_sorted<T, 1>(cand, n, V, out);
    else if (n <= 128) place_sorted<T, 2>(cand, n, V, out);
    else place_sorted<T, 4>(cand, n, V, out);
}

// A workgroup's candidates: by its first wave, or where there are more than 256 by all threads
template <typename T, int TH> __device__ __forceinline__ void place_all(TopLds<TH>& lds, int n, int V, const TopOut& out) {
    if (n <= 256) {
        if (threadIdx.x < 64) place_wave<T>(lds.cand, n, V, out);
        return;
    }
    for (int q = threadIdx.x; q < n; q += TH) {
        const unsigned long long me = lds.cand[q];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) place += lds.cand[j] > me;
        out.write(me, place);
    }
}

// what the gradient takes from a row's sums: m and s, together (one store of a row's 8 bytes costs what each of two costs: rows of a 128-byte line
// come from eight L2s)
typedef __attribute__((ext_vector_type(2), aligned(4))) float row_sums_t;

// (saved: H once more, where the caller may edit `entropy` before the gradient is computed; NULL: not wanted)
template <typename T>
__device__ __forceinline__ void write_row(const T* __restrict__ z, int V, int64_t r, const Acc& a, float inv_t, float log_s, bool empty, const int64_t* __restrict__ tokens,
                                          float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ lse, float* __restrict__ stats, float* __restrict__ saved) {
    *reinterpret_cast<row_sums_t*>(stats + 2 * r) = row_sums_t{a.m, a.s};
    const float h = empty ? 0.f : entropy_of(a, log_s);
    lse[r] = empty ? -INFINITY : a.m * inv_t + log_s;
    entropy[r] = h;
    if (saved) saved[r] = h;
    if (tokens) {
        const int64_t t = tokens[r];
        float v = 0.f;
        if (t >= V) v = NAN;
        else if (t >= 0) v = empty ? -INFINITY : log_prob(Store<T>::load(z + t), a.m, inv_t, log_s);
        logp[r] = v;
    }
}

// parts of rows, for few long ones: `count` workgroups a row, `length` logits each, that leave (m, s, t, -) and k keys to logprobs_join_kernel
struct Parts {
    int count, length;
    float4* acc;
    unsigned long long* keys;
};

// A row, or (PART) one part of it, by TH threads.  Bound by the read of the logits: 16384 x 30522 bf16 in 173 us, 2000 x 32000 fp32 in 40 us
// (5.8 and 6.3 TB/s), with 100 alternatives 8192 x 131072 bf16 in 400 us (6.0 TB/s, 16 % of it the slots that are read again).  A few rows are
// bound by the chain join, bisection, second read, sort: one row of 30522 fp32 with 5 alternatives 10.3 us.  Two chunks a lane are added up
// while two are on their way: four gained nothing and cost a quarter of the waves.
template <typename T, int TH, bool TOP, bool PART>
__global__ __launch_bounds__(TH, 7) void logprobs_wg_kernel(const T* __restrict__ z, int64_t ld, int V, float c, float inv_t, const int64_t* __restrict__ tokens,
                                                         int k, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ lse,
                                                         float* __restrict__ stats, float* __restrict__ saved, int64_t* __restrict__ top_ids,
                                                         float* __restrict__ top_logp, Parts parts) {
    constexpr int E = Chunk<T>::E, U = 2;   // 2 U chunks of a lane are in flight
    __shared__ float red[3 * (TH / 64)];
    const int64_t r = PART ? blockIdx.x / parts.count : blockIdx.x;
    const int base = PART ? blockIdx.x % parts.count * parts.length : 0;
    if (PART) V = min(parts.length, V - base);
    const Row<T> row(z + r * ld + base, V);
    const int tid = threadIdx.x;
    Sums<T, true> sums(c);
    float slot[LG_SLOTS];
#pragma unroll
    for (int i = 0; i < LG_SLOTS; ++i) slot[i] = -INFINITY;
    const int n = row.full(), ei = row.end_index(tid);
    // the next U chunks are on their way while U are added up (loads without a condition: behind the row's end its last chunk again)
    chunk_t v[U], w[U];
    const auto fetch = [&](chunk_t (&to)[U], int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) to[u] = row.load(row.first + min(i0 + u * TH + tid, n - 1));
    };
    fetch(v, 0);
    const float end = ei >= 0 ? Store<T>::load(row.z + ei) : -INFINITY;
    for (int i0 = 0; i0 < n; i0 += LG_SLOTS * TH) {
#pragma unroll
        for (int i = 0; i < LG_SLOTS; i += U) {
            if (i0 + i * TH >= n) break;
            fetch(w, i0 + (i + U) * TH);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + (i + u) * TH + tid < n) {
                    float x[E];
                    Chunk<T>::unpack(v[u], x);
                    const float cmax = max_of(x);
                    if (TOP) slot[i + u] = fmaxf(slot[i + u], cmax);
                    sums.add(x, cmax);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = w[u];
        }
    }
    if (ei >= 0) sums.add_one(end);
    const Acc a = team_join<TH>(sums.acc(), c, red);
    const bool empty = a.s == 0.f;
    const float log_s = empty ? -INFINITY : logf(a.s);
    if (PART) {
        if (tid == 0) parts.acc[blockIdx.x] = make_float4(a.m, a.s, a.t, 0.f);
    } else if (tid == 0) {
        write_row(row.z, V, r, a, inv_t, log_s, empty, tokens, logp, entropy, lse, stats, saved);
    }
    if (!TOP) return;
    __shared__ TopLds<TH> lds;
    constexpr int CAP = TopLds<TH>::CAP;
    if (tid == 0) { lds.n_list = 0; lds.n_cand = 0; }
    uint32_t least;
    if constexpr (TH == 64) {
        float group[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) group[g] = g ? -INFINITY : end;
#pragma unroll
        for (int i = 0; i < LG_SLOTS; ++i) group[i & 3] = fmaxf(group[i & 3], slot[i]);
        least = wave_bound<4, E == 8 ? 16 : 0>(group, k);
    } else {
        float mine[1] = {end};
#pragma unroll
        for (int i = 0; i < LG_SLOTS; ++i) mine[0] = fmaxf(mine[0], slot[i]);
        const uint32_t b = wave_bound<1, E == 8 ? 16 : 0>(mine, (k + TH / 64 - 1) / (TH / 64));
        if ((tid & 63) == 0) lds.bound[tid >> 6] = b;
        __syncthreads();
        least = lds.bound[0];
#pragma unroll
        for (int w = 1; w < TH / 64; ++w) least = min(least, lds.bound[w]);
    }
    const float bound = key_value(least);
    bool whole = a.s != a.s;   // a NaN or +inf in the row
    if (!whole) {
        // (one addition to a counter per lane: its latency is what this part is made of)
        uint32_t which = 0;
#pragma unroll
        for (int i = 0; i < LG_SLOTS; ++i) which |= slot[i] >= bound ? 1u << i : 0u;
        if (which) {
            const int many = __popc(which);
            int at = atomicAdd(&lds.n_list, many);
            if (at + many <= CAP)
                for (; which; which &= which - 1u) lds.list[at++] = (__ffs(which) - 1) * TH + tid;
        }
        if (ei >= 0 && end >= bound) {
            const int at = atomicAdd(&lds.n_cand, 1);
            if (at < CAP) lds.cand[at] = order_key(end, ei);
        }
        Team<TH>::sync();
        const int n_list = lds.n_list, rounds = (n + LG_SLOTS * TH - 1) / (LG_SLOTS * TH);
        whole = n_list > CAP;
        if (!whole) {
            const auto sift = [&](int i, const chunk_t& v) {
                const int lo = (row.first + i) * E - row.sh;
                float x[E];
                Chunk<T>::unpack(v, x);
                uint32_t mine = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) mine |= x[e] >= bound ? 1u << e : 0u;
                const int many = __popc(mine);
                int at = many ? atomicAdd(&lds.n_cand, many) : 0;
                if (at + many <= CAP)
                    for (; mine; mine &= mine - 1u) {
                        const int e = __ffs(mine) - 1;
                        lds.cand[at++] = order_key(Chunk<T>::pick(v, e), lo + e);
                    }
            };
            for (int j = 0; j < rounds; ++j)
                for (int q = tid; q < n_list; q += 2 * TH) {
                    const int i = lds.list[q] + j * (LG_SLOTS * TH), i2 = q + TH < n_list ? lds.list[q + TH] + j * (LG_SLOTS * TH) : n;
                    const chunk_t v = row.load(row.first + min(i, n - 1)), v2 = row.load(row.first + min(i2, n - 1));
                    if (i < n) sift(i, v);
                    if (i2 < n) sift(i2, v2);
                }
            Team<TH>::sync();
            whole = lds.n_cand > CAP;
        }
        Team<TH>::sync();
    }
    if (whole) top_radix<T, TH>(row, k, lds);
    if (PART) place_all<T, TH>(lds, lds.n_cand, V, {nullptr, nullptr, k, 0.f, 0.f, 0.f, false, parts.keys + (int64_t)blockIdx.x * k, base});
    else place_all<T, TH>(lds, lds.n_cand, V, {top_ids + r * k, top_logp + r * k, k, a.m, inv_t, log_s, empty});
}

// One wave a row: its parts' sums (at most 64) and keys (at most 256)
template <typename T, bool TOP>
__global__ __launch_bounds__(64) void logprobs_join_kernel(const T* __restrict__ z, int64_t ld, int V, float c, float inv_t, const int64_t* __restrict__ tokens,
                                                           int k, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ lse,
                                                           float* __restrict__ stats, float* __restrict__ saved, int64_t* __restrict__ top_ids,
                                                           float* __restrict__ top_logp, Parts parts) {
    __shared__ unsigned long long cand[256];
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x, n = parts.count * k;
    if (TOP)
        for (int i = lane; i < n; i += 64) cand[i] = parts.keys[r * n + i];
    const float4 p = parts.acc[r * parts.count + min(lane, parts.count - 1)];
    const Acc mine = {lane < parts.count ? p.x : LG_NEG, lane < parts.count ? p.y : 0.f, lane < parts.count ? p.z : 0.f};
    const Acc a = lanes_join<64>(mine, c);
    const bool empty = a.s == 0.f;
    const float log_s = empty ? -INFINITY : logf(a.s);
    if (lane == 0) write_row(z + r * ld, V, r, a, inv_t, log_s, empty, tokens, logp, entropy, lse, stats, saved);
    Team<64>::sync();
    if (TOP) place_wave<T>(cand, n, V, {top_ids + r * k, top_logp + r * k, k, a.m, inv_t, log_s, empty});
}

// Rows of up to 64 (W = 16 lanes a row) or 2048 logits (W = 64; where a list is long for the row's slots): the whole row lives in registers, the
// maximum is found first.  64000 x 10 fp32 with 3 alternatives 7.8 us, 262144 x 64 129 us: bound by the ranking, which with 16 lanes compares each of
// the row's logits with all of them whatever k is (without alternatives 64000 x 10 takes 4.8 us, of which 0.8 are its bytes).
template <typename T, int W> struct Small;
template <typename T> struct Small<T, 16> {   // element j of a lane: lane + 16 j
    static constexpr int NE = 4;
    static __host__ __device__ constexpr int max_v() { return 16 * NE; }
    const T* z;
    int V, lane;
    __device__ __forceinline__ Small(const T* p, int v, int l) : z(p), V(v), lane(l) {}
    __device__ __forceinline__ int index(int j) const { return lane + 16 * j; }
    template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int j = 0; j < NE; ++j) f(j);
    }
    __device__ __forceinline__ void load(float (&x)[NE]) const {
#pragma unroll
        for (int j = 0; j < NE; ++j) x[j] = index(j) < V ? Store<T>::load(z + index(j)) : -INFINITY;
    }
};
template <typename T> struct Small<T, 64> {   // chunks of a lane: lane + 64 i, and (element NE - 1) one of the row's ends
    static constexpr int E = Chunk<T>::E, NE = 32 + 1, NC = 32 / E;
    static __host__ __device__ constexpr int max_v() { return 64 * 32; }
    Row<T> row;
    int V, lane, end;
    __device__ __forceinline__ Small(const T* p, int v, int l) : row(p, v), V(v), lane(l) { end = row.end_index(l); }
    // the place of element j in the row; of a place the row does not have: -1 or at least V
    __device__ __forceinline__ int index(int j) const { return j == NE - 1 ? end : row_index((j / E) * 64 + lane, j % E); }
    __device__ __forceinline__ int row_index(int i, int e) const { return i < row.full() ? (row.first + i) * E + e - row.sh : V; }
    // f(j) for the lane's elements, chunk rounds that the row does not reach left out
    template <typename F> __device__ __forceinline__ void each_chunk(F f) const {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i * 64 >= row.full()) break;
#pragma unroll
            for (int e = 0; e < E; ++e) f(i * E + e);
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) const {
        each_chunk(f);
        f(NE - 1);
    }
    __device__ __forceinline__ void load(float (&x)[NE]) const {
        const int n = row.full();
        chunk_t v[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = row.load(row.first + min(i * 64 + lane, n - 1));   // (more than 64 logits: n > 0)
        x[NE - 1] = end >= 0 ? Store<T>::load(row.z + end) : -INFINITY;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float y[E];
            Chunk<T>::unpack(v[i], y);
#pragma unroll
            for (int e = 0; e < E; ++e) x[i * E + e] = i * 64 + lane < n ? y[e] : -INFINITY;
        }
    }
};

template <typename T, int W, bool TOP>
__global__ __launch_bounds__(256) void logprobs_small_kernel(const T* __restrict__ z, int64_t ld, int N, int V, float c, float inv_t,
                                                             const int64_t* __restrict__ tokens, int k, float* __restrict__ logp,
                                                             float* __restrict__ entropy, float* __restrict__ lse, float* __restrict__ stats,
                                                             float* __restrict__ saved, int64_t* __restrict__ top_ids, float* __restrict__ top_logp) {
    using S = Small<T, W>;
    constexpr int NE = S::NE, CAP = W == 16 ? 64 : 256;
    const int lane = threadIdx.x & (W - 1), team = threadIdx.x / W;
    const int64_t r = (int64_t)blockIdx.x * (256 / W) + team;
    if (r >= N) return;
    const T* zr = z + r * ld;
    const S row(zr, V, lane);
    float x[NE];
    row.load(x);
    float m = LG_NEG;
#pragma unroll
    for (int j = 0; j < NE; ++j) m = fmaxf(m, x[j]);
    m = lanes_join<W>(m, Max());
    Acc a = {m, 0.f, 0.f};
    row.each([&](int j) {
        const float y = (x[j] - m) * c, p = x[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(y);   // (m may be the type's lowest value)
        a.s += p;
        a.t += p == 0.f ? 0.f : p * y;
    });
    a.s = lanes_join<W>(a.s, Add());
    a.t = lanes_join<W>(a.t, Add());
    const bool empty = a.s == 0.f;
    const float log_s = empty ? -INFINITY : logf(a.s);
    if (lane == 0) write_row(zr, V, r, a, inv_t, log_s, empty, tokens, logp, entropy, lse, stats, saved);
    if (!TOP) return;
    __shared__ unsigned long long cand_lds[256 / W][CAP];
    unsigned long long* cand = cand_lds[team];
    const auto packed = [&](uint32_t key, int i) { return ((unsigned long long)key << 32) | (0xFFFFFFFFu - (uint32_t)i); };
    int n;
    if constexpr (W == 16) {   // every logit is a candidate
        n = V;
        row.each([&](int j) {
            if (row.index(j) < V) cand[row.index(j)] = order_key(x[j], row.index(j));
        });
    } else {
        uint32_t key[NE];
#pragma unroll
        for (int j = 0; j < NE; ++j) key[j] = row.index(j) >= 0 && row.index(j) < V ? order_key(x[j]) : 0u;
        uint32_t at = 0;
        n = V;
        if (V > CAP || V > k + (k >> 1)) {   // (else every logit is a candidate)
            float group[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) group[g] = g ? -INFINITY : x[NE - 1];
            row.each_chunk([&](int j) { group[j & 3] = fmaxf(group[j & 3], x[j]); });
            at = wave_bound<4, Chunk<T>::E == 8 ? 16 : 0>(group, k);
            n = 0;
            row.each([&](int j) { n += __popcll(__ballot(key[j] >= at)); });
        }
        if (n > CAP) {   // equal logits, or a short row's long list: the k-th largest key from the top bit down, until few enough reach it
            at = 0;
            for (int b = 31; b >= 0 && n > CAP; --b) {
                const uint32_t t = at | (1u << b);
                int cnt = 0;
                row.each([&](int j) { cnt += __popcll(__ballot(key[j] >= t)); });
                if (cnt >= k) { at = t; n = cnt; }
            }
        }
        const uint32_t above = n <= CAP ? (at ? at - 1u : 0u) : at;   // (at = 0: every key of the row, they are at least 1)
        const unsigned long long lt = (1ull << lane) - 1ull;
        int out = 0;
        row.each([&](int j) {
            const unsigned long long on = __ballot(key[j] > above);
            if (key[j] > above) cand[out + __popcll(on & lt)] = packed(key[j], row.index(j));
            out += __popcll(on);
        });
        if (n > CAP) {   // many logits equal the k-th: the first of them in the row's order (its head, rounds of chunks by lane and element, its tail)
            int left = k - out;
            const auto take = [&](uint32_t q, int i, bool head) {
                const bool mine = q == at && (lane < Chunk<T>::E) == head;
                const unsigned long long on = __ballot(mine);
                const int before = __popcll(on & lt);
                if (mine && before < left) cand[out + before] = packed(q, i);
                const int took = max(0, min(__popcll(on), left));
                out += took;
                left -= took;
            };
            take(key[NE - 1], row.index(NE - 1), true);
#pragma unroll
            for (int i = 0; i < S::NC; ++i) {
                if (left <= 0) break;
                int before = 0, total = 0;
#pragma unroll
                for (int j = i * S::E; j < i * S::E + S::E; ++j) {
                    const unsigned long long on = __ballot(key[j] == at);
                    before += __popcll(on & lt);
                    total += __popcll(on);
                }
#pragma unroll
                for (int j = i * S::E; j < i * S::E + S::E; ++j)
                    if (key[j] == at) {
                        if (before < left) cand[out + before] = packed(key[j], row.index(j));
                        ++before;
                    }
                const int took = min(total, left);
                out += took;
                left -= took;
            }
            if (left > 0) take(key[NE - 1], row.index(NE - 1), false);
        }
        n = out;
    }
    Team<W>::sync();
    const TopOut result = {top_ids + r * k, top_logp + r * k, k, a.m, inv_t, log_s, empty};
    if constexpr (W == 64) {
        place_wave<T>(cand, n, V, result);
    } else {
        for (int q = lane; q < n; q += W) {
            const unsigned long long me = cand[q];
            int place = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) place += cand[j] > me;
            result.write(me, place);
        }
    }
}

// ---- gradients ------------------------------------------------------------------------------------------------------------------
// Both gradients are one map over the row, e_i = exp2((z_i - m) c) times a number of the row (the entropy's: times a linear function of its
// exponent), and a few places (the given token, the listed ones) where something is added: those are written again once the row is done.
// One read and one write of the row; a lane has U chunks in flight.  Bound by memory: 16384 x 30522 bf16 in 335 us (6.1 TB/s), 2000 x 32000 fp32 in
// 75 us (6.8 TB/s, some of it still cached), with a list of 50 2048 x 65537 bf16 in 84 us (5.9 TB/s).

// Which of a gradient's accesses go past the chip's memory-side cache of 256 MiB.  Logits and gradient that do not fit it together: the stores,
// so that what the forward pass left of the logits stays (what reads the gradient next is a matrix product, which can wait for memory); logits
// that do not fit it alone: the loads too.  Rows of 32001 bf16, forward and backward, a copy into the logits before and a sum of the gradient
// after them taken off: 128 MB of logits 74 us (stores past it: 77), 160 MB 94 -> 86 (loads too: 85), 192 MB 116 -> 99 (103),
// 256 MB 148 -> 129 (124), 300 MB 178 -> 161 (148; without the copy and the sum 181 -> 149, 150), 320 MB 191 -> 177 (159),
// 1 GB 542 -> 530 (518).  The kernel that computes loss and gradient in one gains only where it reads a row twice, and only by the stores: rows of
// 200001 bf16, 100 MB 62 -> 73 us, 160 MB 106 -> 101, 512 MB 278 -> 239, 2 GB 1020 -> 928 (rows of 50001, 410 MB 189 -> 197).
enum Past { PAST_NONE, PAST_STORES, PAST_ALL };
inline Past past_cache(int64_t bytes) {
    constexpr int64_t cache = 256 << 20;
    return bytes <= cache / 2 ? PAST_NONE : bytes <= cache + cache / 8 ? PAST_STORES : PAST_ALL;
}

// What one of gridDim.y workgroups of a row writes of its gradient: a run of chunks, and the row's ends with the first and the last run.
template <typename T> struct Share {
    int lo, hi;   // chunks of the row, counted from the first whole one
    bool head, tail;
    int per, n, to_first;
    __device__ __forceinline__ Share(const Row<T>& row) {
        n = row.full();
        per = (n + (int)gridDim.y - 1) / (int)gridDim.y;
        lo = min((int)blockIdx.y * per, n);
        hi = min(lo + per, n);
        head = blockIdx.y == 0;
        tail = blockIdx.y == gridDim.y - 1;
        to_first = row.first * Row<T>::E - row.sh;
    }
    __device__ __forceinline__ bool has(int i) const {   // logit i of the row
        const int e = i - to_first;
        return e < 0 ? head : e >= n * Row<T>::E ? tail : e >= lo * Row<T>::E && e < hi * Row<T>::E;
    }
};
// f(chunk, its 16 bytes) for a run of the row's chunks, U of a lane at once (loads without a condition, so that all are in flight together:
// behind the run's end its last chunk again)
template <typename T, int TH, int U, Past PAST, typename F> __device__ __forceinline__ void each_chunk(const Row<T>& row, int lo, int hi, F f) {
    const int tid = Team<TH>::rank();
    for (int i0 = lo; i0 < hi; i0 += U * TH) {
        chunk_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ch = row.first + min(i0 + u * TH + tid, hi - 1);
            v[u] = PAST == PAST_ALL ? row.load_past(ch) : row.load(ch);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * TH + tid < hi) f(row.first + i0 + u * TH + tid, v[u]);
    }
}
template <typename T, int TH> __device__ __forceinline__ void zero_row(const Row<T>& row, T* d) {
    constexpr int E = Chunk<T>::E;
    const float x[E] = {};
    const int tid = Team<TH>::rank(), ei = row.end_index(tid);
    if (ei >= 0) Store<T>::store(d + ei, 0.f);
    for (int i = tid; i < row.full(); i += TH) row.store(d, row.first + i, x);
}

// dz_i = inv_t [ p_i (A + B ln p_i) + g_t 1[i = t] + sum_j g_j 1[i = id_j] ],  A = g_lse - g_t - sum_j g_j - g_H H,  B = -g_H
struct LogprobsGrad {
    const float *stats, *entropy, *g_logp, *g_entropy, *g_lse, *g_top;
    const int64_t *tokens, *top_ids;
    int k;
};
template <typename T, int TH, Past PAST>
__global__ __launch_bounds__(TH < 256 ? 256 : TH) void logprobs_bwd_kernel(const T* __restrict__ z, int64_t ld, int N, int V, float c, float inv_t, LogprobsGrad q,
                                                                           T* __restrict__ dz, int64_t ldd) {
    constexpr int E = Chunk<T>::E, U = TH < 64 ? 2 : 4, PER = TH < 256 ? 256 / TH : 1;
    __shared__ float red[TH < 64 ? 1 : TH / 64];
    const int64_t r = (int64_t)blockIdx.x * PER + Team<TH>::index();
    if (PER > 1 && r >= N) return;
    const int tid = Team<TH>::rank();
    const Row<T> row(z + r * ld, V);
    T* d = dz + r * ldd;
    const row_sums_t st = *reinterpret_cast<const row_sums_t*>(q.stats + 2 * r);
    const Acc a = {st.x, st.y, 0.f};
    const int64_t t = q.tokens ? q.tokens[r] : -1;
    const float gt = t < 0 ? 0.f : t < V ? q.g_logp[r] : NAN, gh = q.g_entropy ? q.g_entropy[r] : 0.f;
    float gs = 0.f;
    for (int j = tid; j < q.k; j += TH) gs += q.g_top[r * q.k + j];
    if (q.k) gs = Team<TH>::sum(gs, red);
    const bool empty = a.s == 0.f;
    const float f = empty ? 0.f : inv_t / a.s, log_s = empty ? 0.f : logf(a.s);
    const float A = (q.g_lse ? q.g_lse[r] : 0.f) - gt - gs - gh * q.entropy[r];
    // p (A + B ln p) inv_t = e (c0 + c1 y):  ln p = y ln2 - ln s
    const Ref ref(a.m, c);
    const float undo = __builtin_amdgcn_exp2f(-ref.delta), c1 = undo * -f * gh * LG_LN2, c0 = empty ? 0.f : undo * f * (A + gh * log_s) - c1 * ref.delta;
    const auto one = [&](float x) {
        const float y = fmaxf(ref.y(x, c), -200.f);   // (a masked logit: e = 0, whatever c1 is)
        return __builtin_amdgcn_exp2f(y) * fmaf(c1, y, c0);
    };
    const Share<T> share(row);
    const int ei = row.end_index(tid);
    if (ei >= 0 && share.has(ei)) Store<T>::store(d + ei, one(Store<T>::load(row.z + ei)));
    each_chunk<T, TH, U, PAST>(row, share.lo, share.hi, [&](int ch, const chunk_t& v) {
        float x[E];
        Chunk<T>::unpack(v, x);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = one(x[e]);
        row.template store<PAST != PAST_NONE>(d, ch, x);
    });
    if (empty) return;
    Team<TH>::sync();
    // (top ids are distinct; the given token may be one of them)
    for (int j = tid; j <= q.k; j += TH) {
        const bool is_token = j == q.k;
        const int64_t i = is_token ? t : q.top_ids[r * q.k + j];
        if (i < 0 || i >= V || !share.has((int)i)) continue;
        float g = is_token ? gt : q.g_top[r * q.k + j];
        if (!is_token && i == t) g += gt;
        bool again = false;
        if (is_token)
            for (int p = 0; p < q.k; ++p) again |= q.top_ids[r * q.k + p] == i;
        if (!again) Store<T>::store(d + i, one(Store<T>::load(row.z + i)) + inv_t * g);
    }
}

// ---- distillation ---------------------------------------------------------------------------------------------------------------
// L = tau^2 [ sum_j q_j (ln q_j - ln p_j) + rest (ln rest - ln p_off) ]
// dL/dz_i = tau [ p_i (Q + rest) - q_i - 1[i off the list] rest p_i / p_off ]
// With the tail, the sums over the row leave the listed tokens out (a bit per logit in LDS, set from the list) and the listed ones are added
// from the list: p_off is summed, not the difference of two sums, and holds where the student leaves the rest next to nothing.
struct Distill {
    const int64_t* ids;
    const void* logp;
    int dtype, K;
    const float* weights;
    float weight0;
};

struct Teacher { float Q, rest; };   // the mass on the list, and (with the tail) off it

// a row's list in LDS: token (-1: empty slot, V: no token of the row), mass, its logarithm
struct ListLds {
    int id[AG_LOGITS_MAX_TOP];
    float q[AG_LOGITS_MAX_TOP], lq[AG_LOGITS_MAX_TOP];
};

// The list of a row, by W = 16 or 64 lanes (slots lane + W i): loaded before the row's own loads, and not looked at yet, so that those stay in
// flight while the list is worked on.
template <int W> struct List {
    static constexpr int J = (AG_LOGITS_MAX_TOP + W - 1) / W;
    int64_t raw_id[J];
    uint32_t raw_lp[J];
    static __device__ __forceinline__ int lane() { return threadIdx.x & (W - 1); }
    // f(i) for the rounds of slots that a list of K has
    template <typename F> static __device__ __forceinline__ void each(int K, F f) {
#pragma unroll
        for (int i = 0; i < J; ++i)
            if (i == 0 || i * W < K) f(i);
    }
    __device__ __forceinline__ void load(const Distill& p, int64_t r) {
        each(p.K, [&](int i) {
            const int64_t j = r * p.K + min(lane() + i * W, p.K - 1);
            raw_id[i] = p.ids[j];
            raw_lp[i] = p.dtype == AG_BF16 ? ((const bf16_t*)p.logp)[j] : ((const uint32_t*)p.logp)[j];
        });
    }
    template <bool TAIL> __device__ __forceinline__ Teacher finish(const Distill& p, int V, ListLds& lds) const {
        float lp[J], m = -INFINITY;
        each(p.K, [&](int i) {
            const int j = lane() + i * W;
            const bool there = raw_id[i] >= 0 && j < p.K;
            const int id = !there ? -1 : raw_id[i] >= V ? V : (int)raw_id[i];
            if (j < p.K) lds.id[j] = id;
            lp[i] = !there ? -INFINITY : id == V ? NAN : __uint_as_float(p.dtype == AG_BF16 ? raw_lp[i] << 16 : raw_lp[i]);
            m = fmaxf(m, lp[i]);
        });
        m = lanes_join<W>(m, Max());
        Teacher t = {0.f, 0.f};
        if (!TAIL) {
            float e[J], s = 0.f;
            each(p.K, [&](int i) {
                e[i] = lp[i] == -INFINITY ? 0.f : expf(lp[i] - m);
                s += e[i];
            });
            s = lanes_join<W>(s, Add());
            const float ls = logf(s), is = s == 0.f ? 0.f : 1.f / s;
            each(p.K, [&](int i) {
                const int j = lane() + i * W;
                if (j < p.K) { lds.q[j] = e[i] * is; lds.lq[j] = (lp[i] - m) - ls; }
            });
            t.Q = s == 0.f ? 0.f : s * is;   // (1, or NaN)
        } else {
            float others = 0.f, top = 0.f;   // the masses that are not the largest, and how many are
            each(p.K, [&](int i) {
                const int j = lane() + i * W;
                const float q = lp[i] == -INFINITY ? 0.f : expf(lp[i]);
                if (j < p.K) { lds.q[j] = q; lds.lq[j] = lp[i]; }
                if (lp[i] == m) top += 1.f; else others += q;
            });
            top = lanes_join<W>(top, Add());
            others = lanes_join<W>(others, Add());
            const float q = m == -INFINITY ? 0.f : expf(m);
            t.Q = m == -INFINITY ? others : fmaf(top, q, others);
            // 1 - sum q without the cancellation against its largest term: -expm1 of that one, minus all the others
            t.rest = m == -INFINITY ? 1.f : fmaxf(-expm1f(m) - (top - 1.f) * q - others, 0.f);
            if (t.Q != t.Q) t.rest = t.Q;
        }
        Team<W>::sync();
        return t;
    }
};

// what a row's gradient takes from the forward pass: g a exp2((z - m_off) c) off the list, g (on exp2((z - m) c) - q) on it
struct GradOf { float m_off, a, m, on; };

// The gradients of the listed tokens (W lanes, slots lane + W i; gx: their logits' bits; bit i of `first`: this lane's i-th slot is known to be
// the first that names its token; mine(i): logit i is this workgroup's).  Where a token may be listed more than once its masses are added up: for the
// gradient apart, which knows nothing of the list (`first` 0), always; 131072 x 300 fp32 with lists of 50 takes 156 us, of 128 429, without one 68.
template <typename T, int W, typename F>
__device__ __forceinline__ void listed_gradients(const Row<T>& row, const uint32_t* gx, int K, uint32_t first, const GradOf& s, float g, float c,
                                                 const ListLds& l, T* d, F mine) {
    const int lane = List<W>::lane();
    const auto store = [&](int i, int at, float q) { Store<T>::store(d + at, g * (exp2_from(Row<T>::value(gx[i]), s.m, c) * s.on - q)); };
    uint32_t is = 0;
    List<W>::each(K, [&](int i) { is |= lane + i * W < K && l.id[lane + i * W] >= 0 && l.id[lane + i * W] < row.V ? 1u << i : 0u; });
    if (__any(is != first)) {
        List<W>::each(K, [&](int i) {
            if (!((is >> i) & 1u)) return;
            const int j = lane + i * W, at = l.id[j];
            float q = 0.f;
            bool one = true;
#pragma unroll 4
            for (int o = 0; o < K; ++o) {
                q += l.id[o] == at ? l.q[o] : 0.f;
                one &= l.id[o] != at || o >= j;
            }
            if (one && mine(at)) store(i, at, q);
        });
        return;
    }
    List<W>::each(K, [&](int i) {
        if ((is >> i) & 1u && mine(l.id[lane + i * W])) store(i, l.id[lane + i * W], l.q[lane + i * W]);
    });
}
template <bool PAST, typename T> __device__ __forceinline__ void gradient_chunk(const Row<T>& row, int ch, const chunk_t& v, float c, const Ref& ref, float ga, T* d) {
    constexpr int E = Chunk<T>::E;
    float x[E];
    Chunk<T>::unpack(v, x);
    if (!ref.far) {
        const float gd = ga * __builtin_amdgcn_exp2f(-ref.delta);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = gd * __builtin_amdgcn_exp2f(fmaf(x[e], c, ref.nr));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = ga * exp2_from(x[e], ref.m, c);
    }
    row.template store<PAST>(d, ch, x);
}
// words of LDS for a bit per logit of a row's chunks, whatever its alignment
template <typename T> __host__ __device__ constexpr int bit_words(int V) { return (V + Chunk<T>::E - 1 + 31) / 32 + 1; }

// the row's loss from its sums (off: over what the dense part of the gradient covers, all: over the row), and what its gradient takes from them
template <bool TAIL> __device__ __forceinline__ GradOf row_gradient(const Teacher& tc, const Acc& off, const Acc& all, float c) {
    GradOf s;
    const bool empty = all.s == 0.f;
    s.m_off = off.m;
    s.m = empty ? -INFINITY : all.m;
    s.on = empty ? 0.f : (tc.Q + tc.rest) / all.s;
    s.a = !TAIL ? s.on : off.s == 0.f ? 0.f : s.on * __builtin_amdgcn_exp2f((off.m - all.m) * c) - tc.rest / off.s;
    return s;
}
// kl: the listed tokens' sum of q (ln q - ln p)
template <bool TAIL> __device__ __forceinline__ float row_loss_of(const Teacher& tc, float kl, const Acc& off, const Acc& all, float log_s, float tau, float inv_t) {
    float L = tc.Q != tc.Q ? tc.Q : kl;   // (an id beyond the row)
    if (TAIL && tc.rest != 0.f) L += tc.rest * (logf(tc.rest) - (off.s == 0.f ? -INFINITY : (off.m - all.m) * inv_t + logf(off.s) - log_s));
    return tau * tau * L;
}

// Rows of up to 64 logits, 16 lanes a row: the row, the listed masses of its tokens and the gradient stay in registers.  Bound by the work on the
// lists (each lane looks at every slot).
template <typename T, bool TAIL, bool GRAD>
__global__ __launch_bounds__(256) void distill_small_kernel(const T* __restrict__ z, int64_t ld, int N, int V, float tau, float c, float inv_t, Distill p,
                                                            float* __restrict__ row_loss, float* __restrict__ stats, T* __restrict__ dz, int64_t ldd) {
    using S = Small<T, 16>;
    using G = Team<16>;
    constexpr int NE = S::NE;
    __shared__ ListLds list_lds[16];
    const int team = threadIdx.x / 16, lane = G::rank();
    const int64_t r = (int64_t)blockIdx.x * 16 + team;
    if (r >= N) return;
    T* d = dz + r * ldd;
    const S row(z + r * ld, V, lane);
    const float w = p.weights ? p.weights[r] : p.weight0;
    const bool part = w != 0.f;
    List<16> mine;
    mine.load(p, r);
    float x[NE];
    if (part) row.load(x);
    const ListLds& l = list_lds[team];
    Teacher tc = mine.template finish<TAIL>(p, V, list_lds[team]);
    float q[NE] = {}, qlq = 0.f;   // the masses of the lane's tokens, and of their slots the sum of q ln q
    uint32_t listed = 0;     // bit j: element j is on the list
    for (int j = 0; j < p.K; ++j) {
        const int id = l.id[j];
        const float m = l.q[j], lm = m == 0.f ? 0.f : m * l.lq[j];
#pragma unroll
        for (int e = 0; e < NE; ++e)
            if (id == row.index(e)) { q[e] += m; qlq += lm; listed |= 1u << e; }
    }
    if (TAIL && (int)G::sum((float)__popc(listed), nullptr) >= V && tc.rest == tc.rest) tc.rest = 0.f;   // no token is off the list
    if (!part) {   // the row takes no part
        if (lane == 0) row_loss[r] = 0.f;
        if (!GRAD && lane < 4) stats[r * 4 + lane] = 0.f;
        if (GRAD) row.each([&](int e) { if (row.index(e) < V) Store<T>::store(d + row.index(e), 0.f); });
        return;
    }
    float lm = LG_NEG, om = LG_NEG;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        if (TAIL && !((listed >> e) & 1u)) om = fmaxf(om, x[e]);
        lm = fmaxf(lm, x[e]);
    }
    Acc all = {G::max(lm, nullptr), 0.f, 0.f}, off = {TAIL ? G::max(om, nullptr) : all.m, 0.f, 0.f};
    float ex[NE], so = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const bool on = TAIL && ((listed >> e) & 1u);
        ex[e] = exp2_from(x[e], on ? all.m : off.m, c);
        if (on) all.s += ex[e]; else so += ex[e];
    }
    off.s = G::sum(so, nullptr);
    all.s = TAIL ? G::sum(all.s, nullptr) + rebase(off, all.m, c).s : off.s;
    const bool empty = all.s == 0.f;
    const float log_s = empty ? -INFINITY : logf(all.s);
    float kl = qlq;
#pragma unroll
    for (int e = 0; e < NE; ++e) kl += q[e] == 0.f ? 0.f : q[e] * (empty ? INFINITY : log_s - (x[e] - all.m) * inv_t);
    kl = G::sum(kl, nullptr);
    const GradOf s = row_gradient<TAIL>(tc, off, all, c);
    if (lane == 0) {
        row_loss[r] = row_loss_of<TAIL>(tc, kl, off, all, log_s, tau, inv_t);
        if (!GRAD) *reinterpret_cast<float4*>(stats + r * 4) = make_float4(s.m_off, s.a, s.m, s.on);
    }
    if (!GRAD) return;
    const float g = tau * w;
    row.each([&](int e) {
        if (row.index(e) >= V) return;
        const bool on = (listed >> e) & 1u;
        Store<T>::store(d + row.index(e), empty ? 0.f : on ? g * (ex[e] * s.on - q[e]) : g * s.a * ex[e]);
    });
}

// Loss, and (GRAD) its gradient from the same pass.  A lane holds NC chunks of the row in registers between the sums and the gradient, so a
// row of up to TH NC chunks is read once (a longer one in several rounds, all but the last of them twice).  A row's sums and its gradient
// are work of different kinds with a join between them, and few such rows fit a CU at once: the workgroups stay, and a chunk's registers take
// the next round's or the next row's chunk as soon as the chunk is done with, so that memory is busy through all of it.
// The list is the first wave's: it works on it while the row arrives, marks the listed tokens for the sums of all waves, adds their own part,
// and writes the loss and the listed tokens' gradients.  MULTI: rows of several rounds.
// Bound by memory, reads and writes mixed: 8192 x 131072 bf16 with a list of 100 in 882 us (4.9 TB/s without what the cache gives the second read;
// a copy reaches 4.8), 24576 x 1000 fp32 with 25 in 41 us; the loss alone, 2048 x 65537 bf16 with 50, in 43 us (5.4 TB/s).  Without the prefetch
// in place 8192 x 131072 took 1310 us; 16 rows of 30522 fp32 take 11.2 us, the chain list, sums, join, gradient.
template <typename T, int TH, int NC, bool MULTI, bool TAIL, bool GRAD, Past PAST = PAST_NONE>
__global__ __launch_bounds__(TH < 256 ? 256 : TH, NC == 16 || TH == 1024 ? 4 : NC == 8 ? 5 : 6) void distill_kernel(
    const T* __restrict__ z, int64_t ld, int N, int V, float tau, float c, float inv_t, Distill p, float* __restrict__ row_loss, float* __restrict__ stats,
    T* __restrict__ dz, int64_t ldd) {
    constexpr int E = Chunk<T>::E, PER = TH < 256 ? 256 / TH : 1;
    constexpr int J = List<64>::J, ROUND = NC * TH;
    extern __shared__ uint32_t bits_lds[];
    __shared__ float red[3 * (TH / 64)];
    __shared__ ListLds list_lds[PER];
    __shared__ float said[PER][4];   // the first wave's word: mass on the list, the rest; the listed logits' largest, their exponentials' sum
    const int team = Team<TH>::index(), tid = Team<TH>::rank();
    const bool lead = TH == 64 || __builtin_amdgcn_readfirstlane(tid) < 64;
    const int64_t stride = (int64_t)gridDim.x * PER;
    ListLds& l = list_lds[team];
    uint32_t* bits = bits_lds + team * bit_words<T>(V);   // logit i of the row: bit i + sh, set where it is listed
    for (int i = tid; i < bit_words<T>(V); i += TH) bits[i] = 0u;
    Team<TH>::sync();
    const auto weight = [&](int64_t r) { return p.weights ? scalar_load(p.weights + r) : p.weight0; };
    // the first row from r on that takes part (of those that do not: no loss, no gradient); w: row r's weight, then that row's
    const auto next_row = [&](int64_t r, float& w) {
        for (; r < N && w == 0.f; w = weight(min(r += stride, (int64_t)N - 1))) {
            if (tid == 0) row_loss[r] = 0.f;
            if (!GRAD && tid < 4) stats[r * 4 + tid] = 0.f;
            if (GRAD) zero_row<T, TH>(Row<T>(z + r * ld, V), dz + r * ldd);
        }
        return r;
    };
    int64_t r = (int64_t)blockIdx.x * PER + team;
    if (r >= N) return;
    float w = weight(r);
    r = next_row(r, w);
    if (r >= N) return;
    float w2 = weight(min(r + stride, (int64_t)N - 1));
    List<64> mine;
    chunk_t v[NC];
    if (lead) mine.load(p, r);
    Row<T> row(z + r * ld, V);
    // (of the logits at a row's ends: the bits, read whether the thread has one or not)
    uint32_t end = row.bits(max(row.end_index(tid), 0));
    {
        const int last = row.full() - 1;
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = row.load(row.first + min(i * TH + tid, last));
    }
    for (;;) {
        // (the places of a thread's chunks are worked out where they are used, from a number that the compiler cannot see through: kept over
        // the loop, they are NC registers that the chunks themselves need)
        int t0 = tid, t1 = tid;
        asm volatile("" : "+v"(t0));
        const int n = row.full();
        T* d = dz + r * ldd;
        const int64_t r2 = next_row(r + stride, w2);
        const float w3 = weight(min(r2 + stride, (int64_t)N - 1));
        const Row<T> row2(r2 < N ? z + r2 * ld : row.z, V);
        const int last2 = r2 < N ? row2.full() - 1 : 0;   // (no next row: its loads are one chunk of this one, again and again)
        Teacher tc = {0.f, 0.f};
        uint32_t gx[J];   // the slots' tokens' logits
        uint32_t first = 0;    // bit i: this lane's i-th slot names a token that no earlier one does
        int at[J] = {};
        uint32_t again = 0;
        if (lead) {
            tc = mine.template finish<TAIL>(p, V, l);
            List<64>::each(p.K, [&](int i) {
                const int id = tid + i * 64 < p.K ? l.id[tid + i * 64] : -1;
                if (id < 0 || id >= V) return;
                at[i] = id;
                const uint32_t b = 1u << ((id + row.sh) & 31);
                if (!(atomicOr(&bits[(id + row.sh) >> 5], b) & b)) first |= 1u << i;
                else again = 1u;
            });
            if (__any(again)) {   // a token listed twice: its first slot is the lower one, whichever came first just now
                first = 0;
                List<64>::each(p.K, [&](int i) {
                    const int j = tid + i * 64, id = j < p.K ? l.id[j] : -1;
                    bool is = id >= 0 && id < V;
                    for (int o = 0; o < p.K; ++o) is &= l.id[o] != id || o >= j;
                    if (is) first |= 1u << i;
                });
            }
            if (TAIL && TH == 64 && (int)lanes_join<64>((float)__popc(first), Add()) == V && tc.rest == tc.rest) tc.rest = 0.f;   // no token is off the list
            if (TH > 64 && tid == 0) { said[team][0] = tc.Q; said[team][1] = tc.rest; }
        }
        List<64>::each(p.K, [&](int i) { gx[i] = row.bits(at[i]); });   // (by all waves: a load that nothing waits for)
        if (TAIL) Team<TH>::sync();
        Sums<T, false> sums(c);
        const auto add_chunk = [&](int i, int ch) {
            float y[E];
            Chunk<T>::unpack(v[i], y);
            if (TAIL) {
                const uint8_t* byte = reinterpret_cast<const uint8_t*>(bits);
                const uint32_t b = E == 8 ? byte[ch] : (byte[ch >> 1] >> ((ch & 1) * 4)) & 15u;
                if (b) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if ((b >> e) & 1u) y[e] = -INFINITY;
                }
            }
            sums.add(y, max_of(y));
        };
        const int lastr = MULTI ? (n - 1) / ROUND * ROUND : 0;
        for (int i0 = 0; i0 < lastr; i0 += ROUND) {
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                add_chunk(i, row.first + i0 + i * TH + t0);
                v[i] = row.load(row.first + min(i0 + ROUND + i * TH + t0, n - 1));
            }
        }
        uint32_t end2 = 0;
        if (!GRAD) {
            if (lead) mine.load(p, r2 < N ? r2 : r);
            end2 = row2.bits(max(row2.end_index(tid), 0));
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            asm volatile("" : "+v"(v[i]));   // (waited for whether it is added or not: the compiler then knows that all have come in)
            if (lastr + i * TH + t0 < n) add_chunk(i, row.first + lastr + i * TH + t0);
            if (!GRAD) v[i] = row2.load(row2.first + min(i * TH + t0, last2));
        }
        const int ei = row.end_index(tid);
        if (ei >= 0 && !(TAIL && (bits[(ei + row.sh) >> 5] >> ((ei + row.sh) & 31) & 1u))) sums.add_one(Row<T>::value(end));
        Acc listed = {LG_NEG, 0.f, 0.f};
        if (TAIL && lead) {   // the listed tokens' part of the sums
            List<64>::each(p.K, [&](int i) { listed.m = fmaxf(listed.m, (first >> i) & 1u ? Row<T>::value(gx[i]) : LG_NEG); });
            listed.m = lanes_join<64>(listed.m, Max());
            List<64>::each(p.K, [&](int i) { listed.s += (first >> i) & 1u ? exp2_from(Row<T>::value(gx[i]), listed.m, c) : 0.f; });
            listed.s = lanes_join<64>(listed.s, Add());
            if (TH > 64 && tid == 0) { said[team][2] = listed.m; said[team][3] = listed.s; }
        }
        const Acc off = team_join<TH>(sums.acc(), c, red);
        if (TH > 64) {
            tc = {said[team][0], said[team][1]};
            if (TAIL) listed = {said[team][2], said[team][3], 0.f};
        }
        Acc all = off;
        if (TAIL) {
            const float m = fmaxf(off.m, listed.m);
            all = rebase(off, m, c);
            all.s += rebase(listed, m, c).s;
        }
        const bool empty = all.s == 0.f;
        const GradOf s = row_gradient<TAIL>(tc, off, all, c);
        if (lead) {
            const float log_s = empty ? -INFINITY : logf(all.s);
            float kl = 0.f;
            List<64>::each(p.K, [&](int i) {
                const int j = tid + i * 64;
                const float q = j < p.K ? l.q[j] : 0.f;
                kl += q == 0.f ? 0.f : q * (empty ? INFINITY : l.lq[j] + log_s - (Row<T>::value(gx[i]) - all.m) * inv_t);
                if (j < p.K && l.id[j] >= 0 && l.id[j] < V) bits[(l.id[j] + row.sh) >> 5] = 0u;   // (every wave is done with them)
            });
            kl = lanes_join<64>(kl, Add());
            if (tid == 0) {
                row_loss[r] = row_loss_of<TAIL>(tc, kl, off, all, log_s, tau, inv_t);
                if (!GRAD) *reinterpret_cast<float4*>(stats + r * 4) = make_float4(s.m_off, s.a, s.m, s.on);
            }
        }
        if (GRAD) {
            if (lead) mine.load(p, r2 < N ? r2 : r);
            end2 = row2.bits(max(row2.end_index(tid), 0));
            const Ref ref(s.m_off, c);
            const float g = tau * w, ga = empty ? 0.f : g * s.a;
            asm volatile("" : "+v"(t1));
            if (ei >= 0) Store<T>::store(d + ei, ga * exp2_from(Row<T>::value(end), ref.m, c));
            // the last round's chunks are still here; the rounds before it, then the next row's first round come in their places
            const auto round = [&](int i0, bool again) {
                const T* from = again ? row.z + ((row.first + i0 - ROUND) * E - row.sh) : row2.z + (row2.first * E - row2.sh);
                const int to = again ? ROUND - 1 : last2;
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    // (a new value for the compiler: else it keeps the sums' unpacked logits, twice the chunks' registers, for the gradient)
                    asm volatile("" : "+v"(v[i]));
                    if (i0 + i * TH + t1 < n) gradient_chunk<PAST != PAST_NONE>(row, row.first + i0 + i * TH + t1, v[i], c, ref, ga, d);
                    v[i] = *reinterpret_cast<const chunk_t*>(from + min(i * TH + t1, to) * E);
                }
            };
            if (!MULTI) round(0, false);
            else
                for (int i0 = lastr; i0 >= 0; i0 -= ROUND) round(i0, i0 > 0);
            Team<TH>::sync();
            if (lead && !empty) listed_gradients<T, 64>(row, gx, p.K, first, s, g, c, l, d, [](int) { return true; });
        } else {
            Team<TH>::sync();   // (the first wave's words are read)
        }
        if (r2 >= N) break;
        r = r2;
        w = w2;
        w2 = w3;
        row = row2;
        end = end2;
    }
}

// The gradient apart from the loss: the same map and list, with the row's numbers read back.
template <typename T, int TH, bool TAIL, Past PAST>
__global__ __launch_bounds__(TH < 256 ? 256 : TH) void distill_bwd_kernel(const T* __restrict__ z, int64_t ld, int N, int V, float tau, float c, Distill p,
                                                                          const float* __restrict__ stats, const float* __restrict__ g_loss,
                                                                          const float* __restrict__ g_row, T* __restrict__ dz, int64_t ldd) {
    constexpr int U = TH < 64 ? 2 : 4, PER = TH < 256 ? 256 / TH : 1, W = TH < 64 ? TH : 64;
    __shared__ ListLds list_lds[PER];
    const int team = Team<TH>::index(), tid = Team<TH>::rank();
    const bool lead = TH <= 64 || __builtin_amdgcn_readfirstlane(tid) < 64;
    const int64_t r = (int64_t)blockIdx.x * PER + team;
    if (PER > 1 && r >= N) return;
    const Row<T> row(z + r * ld, V);
    T* d = dz + r * ldd;
    const float w = p.weights ? p.weights[r] : p.weight0;
    const float4 st = *reinterpret_cast<const float4*>(stats + r * 4);
    const GradOf s = {st.x, st.y, st.z, st.w};
    const Share<T> share(row);
    if (w == 0.f || s.m == -INFINITY) {   // the row takes no part, or none of its logits is above -inf
        if (share.head) zero_row<T, TH>(row, d);
        return;
    }
    List<W> mine;
    if (lead) mine.load(p, r);
    const Ref ref(s.m_off, c);
    const float g = tau * (g_loss || g_row ? (g_loss ? w * g_loss[0] : 0.f) + (g_row ? g_row[r] : 0.f) : w);
    const float ga = g * s.a;
    const int ei = row.end_index(tid);
    if (ei >= 0 && share.has(ei)) Store<T>::store(d + ei, ga * exp2_from(Store<T>::load(row.z + ei), ref.m, c));
    each_chunk<T, TH, U, PAST>(row, share.lo, share.hi, [&](int ch, const chunk_t& v) { gradient_chunk<PAST != PAST_NONE>(row, ch, v, c, ref, ga, d); });
    uint32_t gx[List<W>::J];
    if (lead) {
        mine.template finish<TAIL>(p, V, list_lds[team]);
        List<W>::each(p.K, [&](int i) { gx[i] = row.bits(min(max(list_lds[team].id[min(tid + i * W, p.K - 1)], 0), V - 1)); });
    }
    Team<TH>::sync();
    if (lead) listed_gradients<T, W>(row, gx, p.K, 0u, s, g, c, list_lds[team], d, [&](int i) { return share.has(i); });
}

// sum_n w_n L_n in a fixed order, in doubles (a product of two floats is exact): one workgroup, latency: 16 rows 2.5 us, 24576 4.0,
// 200000 24 (more loads in flight, 16 or 24 of each array: the same; one wave for few rows: 2.1 us)
__global__ __launch_bounds__(1024) void weighted_sum_kernel(const float* __restrict__ row_loss, const float* __restrict__ weights, float weight0, int N,
                                                            float* __restrict__ loss) {
    __shared__ double red[16];
    double acc = 0.0;
    for (int i0 = threadIdx.x; i0 < N; i0 += 8 * 1024) {   // (eight loads of each array in flight)
        float w[8], v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = min(i0 + u * 1024, N - 1);
            w[u] = weights ? weights[i] : weight0;
            v[u] = row_loss[i];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * 1024 < N && w[u] != 0.f) acc += (double)w[u] * (double)v[u];
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

// ---- host -----------------------------------------------------------------------------------------------------------------------
int check_rows(const char* who, const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature) {
    AG_REQUIRE(N >= 0 && V >= 1 && V <= AG_LOGITS_MAX_V, "%s: %d rows x %d logits (1 to %d logits per row)", who, N, V, AG_LOGITS_MAX_V);
    AG_REQUIRE(d_logits || N == 0, "%s: null pointer", who);
    AG_REQUIRE(dtype == AG_F32 || dtype == AG_BF16, "%s: dtype %d (AG_F32 or AG_BF16)", who, dtype);
    AG_REQUIRE(ld >= 0, "%s: row stride %lld", who, (long long)ld);
    AG_REQUIRE(temperature >= 0x1p-20f && temperature <= 0x1p20f, "%s: temperature %g (2^-20 to 2^20)", who, (double)temperature);
    // (a launch holds less than 2^32 threads; at most this many belong to a row)
    const int chunks = V / (dtype == AG_BF16 ? 8 : 4), threads = V <= 64 ? 16 : chunks <= 320 ? 64 : chunks <= 2048 ? 256 : 1024;
    AG_REQUIRE((int64_t)N * threads < (int64_t)1 << 32, "%s: %d rows of %d logits in one call (fewer than %lld)", who, N, V,
               ((long long)1 << 32) / threads);
    return AG_OK;
}
int check_teacher(const char* who, const void* ids, const void* t_logp, int t_dtype, int K, int N) {
    AG_REQUIRE(K >= 1 && K <= AG_LOGITS_MAX_TOP, "%s: lists of %d tokens (1 to %d)", who, K, AG_LOGITS_MAX_TOP);
    AG_REQUIRE(N == 0 || (ids && t_logp), "%s: null pointer", who);
    AG_REQUIRE(t_dtype == AG_F32 || t_dtype == AG_BF16, "%s: teacher dtype %d (AG_F32 or AG_BF16)", who, t_dtype);
    return AG_OK;
}
float log2e_over(float temperature) { return (float)(1.4426950408889634074 / (double)temperature); }
float one_over(float temperature) { return (float)(1.0 / (double)temperature); }

// The gradients' launches, by the row's 16-byte pieces and by the rows a CU gets (log-probabilities' gradient, fp32, both sides of each bound):
//   up to 32: 16 lanes a row          131072 rows of 128: 23.6 us, 64 lanes 53.6; of 300: 68.0 / 76.8 (with a list of 50: 168.8 / 146.1)
//   up to 320: 64 lanes               65536 rows of 1200: 124 us, 256 threads 137; of 1600: 159 / 151
//   up to one row a CU, longer: several workgroups of 256 threads a row, at least 1024 pieces each
//                                     one row of 262144: 5.0 us, one workgroup 22.1; 256 rows of 131072: 41 / 44
//   up to 2048: 256 threads           16384 rows of 6000: 151 us, 1024 threads 160; of 8192: 199 / 192; 8192 of 16384: 207 / 188
//   longer: 1024 threads
#define LG_GRADIENT(V, N, CALL)                                                                                                    \
    const int row_chunks = (V) / Chunk<T>::E;                                                                                      \
    if (row_chunks <= 32) { CALL(16, 1); }                                                                                         \
    else if (row_chunks <= 320) { CALL(64, 1); }                                                                                   \
    else if ((N) <= cu_count()) { CALL(256, std::max(1, std::min(8 * cu_count() / (N), row_chunks / 1024))); }                     \
    else if (row_chunks <= 2048) { CALL(256, 1); }                                                                                 \
    else { CALL(1024, 1); }
int cu_count() { return ag_device_cus() > 0 ? ag_device_cus() : 256; }
template <int TH> dim3 team_grid(int N, int y = 1) { return dim3(TH < 256 ? ceil_div(N, 256 / TH) : N, y); }

// How many workgroups share a row: up to 128 rows of 32768 chunks and more, as many as the join takes (64 sums, 256 keys), as give each CU two
// and leave each 1024 chunks (256 threads, four rounds).  Kernels alone, N x V fp32, k alternatives, shared / one workgroup a row: 1 x 131072,
// k 0: 8.5 / 13.0 us, k 16: 13.8 / 20.2; 1 x 524288, k 4: 13.6 / 50.5; 128 x 131072, k 16: 20.9 / 23.6.  Not for more than 32 alternatives,
// which leave the join of 256 keys few parts (1 x 131072, k 64: 20.9 / 22.0, k 128: 29.7 / 22.5; longer rows were not measured so: there one workgroup
// is 50 us of a call of 1 x 524288 with k 33 to 64, where k 32, shared, is 28), nor for shorter rows (1 x 65536, k 16: 14.3 / 14.3): the second launch and
// the workspace cost the host 5 us.
// (The last part has what the rounding up to 64 logits leaves it: at least 4096 - 63 * 64 logits, and at least k.)
Parts parts_of(int N, int V, int dtype, int k) {
    const int chunks = V / (dtype == AG_BF16 ? 8 : 4);
    if (N < 1 || N > AG_LOGITS_SHARED_ROWS || chunks < AG_LOGITS_SHARED_PIECES || V > AG_LOGITS_MAX_V || k < 0 || k > 32 || (dtype != AG_F32 && dtype != AG_BF16)) return {0, 0, nullptr, nullptr};
    const int count = std::min(std::min(64, chunks / 1024), std::min(k ? 256 / k : 64, 512 / N));
    const int length = (ceil_div(V, count) + 63) / 64 * 64;
    return {ceil_div(V, length), length, nullptr, nullptr};
}

// Threads of a row, by its chunks and the rows a CU gets (N rows of V logits, k alternatives, both sides of each bound):
//   V <= 64: 16 lanes                        262144 x 64 fp32, k 3: 129 us, 64 lanes 282
//   up to 2048 chunks: 64 lanes              16384 x 6000 fp32, k 20: 78 us, 256 threads 90; x 8192: 109 / 104 (bf16 x 16384: 111 / 118)
//       four rows a CU or fewer: up to 512   512 x 4096 bf16, k 50: 11.0 / 9.7 us; 64 x 16384: 17.1 / 10.5; 1024 x 2080: 10.1 / 11.4
//   up to 8192: 256 threads                  8192 x 32768 bf16, k 20: 103 us, 512 threads 132; 2048 x 65536 fp32, k 100: 112 / 107
//       one row a CU or fewer: up to 4096    1 x 32000 fp32, k 16: 12.2 / 9.8 us; 256 x 16000: 10.3 / 10.5
//   longer: 512 threads
//       one row a CU or fewer, longer than 16384: 1024 threads      64 x 240000 fp32, k 128: 35.7 us, 512 threads 42.0; x 65536: 20.3 / 20.1
template <typename T, bool TOP>
int logprobs(const void* d_logits, int64_t ld, int N, int V, float temperature, const int64_t* d_tokens, int k, float* d_logp, float* d_entropy, float* d_lse,
             float* d_stats, float* d_saved, int64_t* d_top_ids, float* d_top_logp, Parts parts, hipStream_t s) {
    const float c = log2e_over(temperature), inv_t = one_over(temperature);
    const T* z = (const T*)d_logits;
#define LG_SMALL(W) hipLaunchKernelGGL((logprobs_small_kernel<T, W, TOP>), team_grid<W>(N), dim3(256), 0, s, z, ld, N, V, c, inv_t, d_tokens, k, d_logp, \
                                       d_entropy, d_lse, d_stats, d_saved, d_top_ids, d_top_logp)
#define LG_WG(TH, PART) hipLaunchKernelGGL((logprobs_wg_kernel<T, TH, TOP, PART>), dim3(N * (PART ? parts.count : 1)), dim3(TH), 0, s, z, ld, V, c, inv_t, \
                                           d_tokens, k, d_logp, d_entropy, d_lse, d_stats, d_saved, d_top_ids, d_top_logp, parts)
    const int chunks = V / Chunk<T>::E, cus = cu_count();
    if (parts.count) {
        LG_WG(256, true);
        AG_LAUNCH_CHECK();
        hipLaunchKernelGGL((logprobs_join_kernel<T, TOP>), dim3(N), dim3(64), 0, s, z, ld, V, c, inv_t, d_tokens, k, d_logp, d_entropy, d_lse, d_stats,
                           d_saved, d_top_ids, d_top_logp, parts);
    } else if (V <= Small<T, 16>::max_v()) LG_SMALL(16);
    else if (V <= Small<T, 64>::max_v() && (chunks < 16 || min(chunks, 64 * min(max(chunks / 64, 1), 4)) < k + k / 2)) LG_SMALL(64);
    else if (chunks <= (N <= 4 * cus ? 512 : 2048)) LG_WG(64, false);
    else if (chunks <= (N <= cus ? 4096 : 8192)) LG_WG(256, false);
    else if (N <= cus && chunks > 16384) LG_WG(1024, false);
    else LG_WG(512, false);
#undef LG_SMALL
#undef LG_WG
    AG_LAUNCH_CHECK();
    return AG_OK;
}

template <typename T>
int logprobs_bwd(const void* d_logits, int64_t ld, int N, int V, float temperature, const LogprobsGrad& q, void* d_dlogits, int64_t ldd, hipStream_t s) {
    const Past past = past_cache((int64_t)N * V * (int64_t)sizeof(T));
#define LG_CALL(TH, Y)                                                                                                                                \
    const auto kernel = past == PAST_NONE     ? logprobs_bwd_kernel<T, TH, PAST_NONE>                                                                 \
                        : past == PAST_STORES ? logprobs_bwd_kernel<T, TH, PAST_STORES>                                                               \
                                              : logprobs_bwd_kernel<T, TH, PAST_ALL>;                                                                 \
    hipLaunchKernelGGL(kernel, team_grid<TH>(N, Y), dim3(TH < 256 ? 256 : TH), 0, s, (const T*)d_logits, ld, N, V, log2e_over(temperature),           \
                       one_over(temperature), q, (T*)d_dlogits, ldd)
    LG_GRADIENT(V, N, LG_CALL)
#undef LG_CALL
    AG_LAUNCH_CHECK();
    return AG_OK;
}

// Threads of a row and chunks of a thread: the fewest threads whose registers hold the row.  With the gradient, 16384 rows fp32, list of 50,
// the choice against its neighbour: V 1000: (64, 4) 43.6 us, (64, 8) 50.0; 2040: (64, 8) 80.8, (256, 8) 118.6; 2400: (64, 16) 90, (256, 8) 118;
// 4000: 141 / 143; 8160: (256, 8) 248, (256, 16) 254; 11184 x 12000: (256, 16) 248, (512, 16) 258; 5592 x 24000: (512, 16) 233, (1024, 16) 274;
// 2048 x 65520: one round of (1024, 16) 245, rounds of (256, 8) 293; past the cache two rounds of (512, 16) instead, the second read being the cache's and
// two workgroups a CU taking turns.  bf16 rows of 72001 / 96001 / 130401, list of 64 + rest, two rounds / one: 140 MB 74 / 77, 63 / 77, 65 / 89 us; 300 MB
// 158 / 166, 143 / 167, 131 / 159; 500 MB 259 / 250, 239 / 252, 237 / 250; 1 GB 498 / 482, 456 / 463, 458 / 463; 2 GB 973 / 926, 897 / 889, 912 / 895, but
// 8192 x 131072 (2.1 GB, aligned rows) 882 / 918.  Four rows a CU or fewer are a matter of latency: 512 x 2040: (64, 8) 11.7, (256, 8) 10.6; 64 x 16360:
// (256, 16) 13.8, (512, 16) 12.0.
// The loss alone reads each chunk once, whatever the rounds: 8388 x 4000: (64, 4) 32.3, (256, 4) 43.6; 2796 x 12000: 27.5 / 29.7; 2048 x 16384:
// 29.1 / 27.9; 512 x 4000: 10.7 / 9.1; one row a CU or fewer, 64 x 64000: (256, 4) 20.1, (1024, 8) 13.0.
template <typename T, bool TAIL, bool GRAD>
int distill(const void* d_logits, int64_t ld, int N, int V, float temperature, const Distill& p, float* d_row_loss, float* d_stats, void* d_dlogits,
            int64_t ldd, hipStream_t s) {
    const T* z = (const T*)d_logits;
    T* dz = (T*)d_dlogits;
    const float c = log2e_over(temperature), inv_t = one_over(temperature);
    const int chunks = V / Chunk<T>::E, cus = cu_count();
    if (V <= Small<T, 16>::max_v()) {
        hipLaunchKernelGGL((distill_small_kernel<T, TAIL, GRAD>), dim3(ceil_div(N, 16)), dim3(256), 0, s, z, ld, N, V, temperature, c, inv_t, p, d_row_loss,
                           d_stats, dz, ldd);
        AG_LAUNCH_CHECK();
        return AG_OK;
    }
#define LG_CALL(TH, NC, MULTI, PER_CU, ...)                                                                                                                       \
    hipLaunchKernelGGL((distill_kernel<T, TH, NC, MULTI, TAIL, GRAD __VA_OPT__(, ) __VA_ARGS__>), dim3(min(ceil_div(N, TH < 256 ? 256 / TH : 1), cus * (PER_CU))), dim3(TH < 256 ? 256 : TH), \
                       (size_t)bit_words<T>(V) * 4 * (TH < 256 ? 256 / TH : 1), s, z, ld, N, V, temperature, c, inv_t, p, d_row_loss, d_stats, dz, ldd)
    if constexpr (GRAD) {
        if (chunks <= 4 * 64) LG_CALL(64, 4, false, 6);
        else if (N > 4 * cus && chunks <= 8 * 64) LG_CALL(64, 8, false, 5);
        else if (N > 4 * cus && chunks <= 16 * 64) LG_CALL(64, 16, false, 4);
        else if (chunks <= 8 * 256) LG_CALL(256, 8, false, 5);
        else if (N > 2 * cus && chunks <= 16 * 256) LG_CALL(256, 16, false, 4);
        else if (chunks <= 16 * 512) LG_CALL(512, 16, false, 2);
        else if (past_cache((int64_t)N * V * (int64_t)sizeof(T)) == PAST_NONE) {
            if (chunks <= 16 * 1024) LG_CALL(1024, 16, false, 1);
            else LG_CALL(1024, 16, true, 1);
        } else {
            if (chunks <= 16 * 1024) LG_CALL(512, 16, true, 2, PAST_STORES);
            else LG_CALL(1024, 16, true, 1, PAST_STORES);
        }
    } else {
        if (chunks <= (N <= 4 * cus ? 512 : 2048)) LG_CALL(64, 4, true, 6);
        else if (N <= cus && chunks >= 4096) LG_CALL(1024, 8, true, 1);
        else LG_CALL(256, 4, true, 6);
    }
#undef LG_CALL
    AG_LAUNCH_CHECK();
    return AG_OK;
}

template <typename T, bool TAIL>
int distill_bwd(const void* d_logits, int64_t ld, int N, int V, float temperature, const Distill& p, const float* d_stats, const float* d_g_loss,
                const float* d_g_row, void* d_dlogits, int64_t ldd, hipStream_t s) {
    const Past past = past_cache((int64_t)N * V * (int64_t)sizeof(T));
#define LG_CALL(TH, Y)                                                                                                                                \
    const auto kernel = past == PAST_NONE     ? distill_bwd_kernel<T, TH, TAIL, PAST_NONE>                                                            \
                        : past == PAST_STORES ? distill_bwd_kernel<T, TH, TAIL, PAST_STORES>                                                          \
                                              : distill_bwd_kernel<T, TH, TAIL, PAST_ALL>;                                                            \
    hipLaunchKernelGGL(kernel, team_grid<TH>(N, Y), dim3(TH < 256 ? 256 : TH), 0, s, (const T*)d_logits, ld, N, V, temperature,                       \
                       log2e_over(temperature), p, d_stats, d_g_loss, d_g_row, (T*)d_dlogits, ldd)
    LG_GRADIENT(V, N, LG_CALL)
#undef LG_CALL
    AG_LAUNCH_CHECK();
    return AG_OK;
}

auto gradient_of(int dtype, int tail) {
    return dtype == AG_BF16 ? (tail ? distill_bwd<bf16_t, true> : distill_bwd<bf16_t, false>) : (tail ? distill_bwd<float, true> : distill_bwd<float, false>);
}

}  // namespace

extern "C" size_t ag_token_logprobs_workspace_bytes(int N, int V, int dtype, int top_k) {
    const Parts p = parts_of(N, V, dtype, top_k);
    return p.count ? (size_t)N * p.count * (sizeof(float4) + (size_t)top_k * sizeof(unsigned long long)) : 0;
}

static int token_logprobs_entry(const char* who, const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_tokens, int top_k,
                                float* d_logp, float* d_entropy, float* d_lse, float* d_stats, float* d_saved, int64_t* d_top_ids, float* d_top_logp,
                                void* d_workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_rows(who, d_logits, ld, N, V, dtype, temperature)) return rc;
    AG_REQUIRE(top_k >= 0 && top_k <= AG_LOGITS_MAX_TOP && top_k <= V, "%s: top_k = %d (0 to min(%d, %d logits))", who, top_k, AG_LOGITS_MAX_TOP, V);
    if (N == 0) return AG_OK;
    AG_REQUIRE(d_entropy && d_lse && d_stats && (!d_tokens || d_logp) && (top_k == 0 || (d_top_ids && d_top_logp)), "%s: null pointer", who);
    const size_t need = ag_token_logprobs_workspace_bytes(N, V, dtype, top_k);
    AG_REQUIRE(!d_workspace || (workspace_bytes >= need && ((uintptr_t)d_workspace & 15) == 0), "%s: workspace of %zu bytes (16-byte aligned, %zu needed)", who,
               workspace_bytes, need);
    Parts parts = {0, 0, nullptr, nullptr};
    if (d_workspace && need) {
        parts = parts_of(N, V, dtype, top_k);
        parts.acc = (float4*)d_workspace;
        parts.keys = (unsigned long long*)(parts.acc + (size_t)N * parts.count);
    }
    const auto run = dtype == AG_BF16 ? (top_k ? logprobs<bf16_t, true> : logprobs<bf16_t, false>) : (top_k ? logprobs<float, true> : logprobs<float, false>);
    return run(d_logits, ld, N, V, temperature, d_tokens, top_k, d_logp, d_entropy, d_lse, d_stats, d_saved, d_top_ids, d_top_logp, parts, (hipStream_t)stream);
}

extern "C" int ag_token_logprobs(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_tokens, int top_k,
                                 float* d_logp, float* d_entropy, float* d_lse, float* d_stats, int64_t* d_top_ids, float* d_top_logp,
                                 void* d_workspace, size_t workspace_bytes, void* stream) {
    return token_logprobs_entry("ag_token_logprobs", d_logits, ld, N, V, dtype, temperature, d_tokens, top_k, d_logp, d_entropy, d_lse, d_stats, nullptr, d_top_ids,
                                d_top_logp, d_workspace, workspace_bytes, stream);
}

extern "C" int ag_token_logprobs_saved(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_tokens, int top_k,
                                       float* d_logp, float* d_entropy, float* d_lse, float* d_stats, float* d_saved_entropy, int64_t* d_top_ids,
                                       float* d_top_logp, void* d_workspace, size_t workspace_bytes, void* stream) {
    AG_REQUIRE(d_saved_entropy || N == 0, "ag_token_logprobs_saved: null pointer");
    return token_logprobs_entry("ag_token_logprobs_saved", d_logits, ld, N, V, dtype, temperature, d_tokens, top_k, d_logp, d_entropy, d_lse, d_stats,
                                d_saved_entropy, d_top_ids, d_top_logp, d_workspace, workspace_bytes, stream);
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
    const LogprobsGrad q = {d_stats, d_entropy, d_g_logp, d_g_entropy, d_g_lse, d_g_top_logp, d_g_logp ? d_tokens : nullptr, d_top_ids,
                            d_g_top_logp ? top_k : 0};
    return (dtype == AG_BF16 ? logprobs_bwd<bf16_t> : logprobs_bwd<float>)(d_logits, ld, N, V, temperature, q, d_dlogits, ldd, (hipStream_t)stream);
}

extern "C" int ag_topk_distill(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_teacher_ids,
                               const void* d_teacher_logp, int teacher_dtype, int K, const float* d_weights, int tail, float* d_row_loss,
                               float* d_loss, float* d_stats, void* d_dlogits, int64_t ldd, void* stream) {
    if (int rc = check_rows("ag_topk_distill", d_logits, ld, N, V, dtype, temperature)) return rc;
    if (int rc = check_teacher("ag_topk_distill", d_teacher_ids, d_teacher_logp, teacher_dtype, K, N)) return rc;
    AG_REQUIRE(N >= 1 && d_row_loss && d_loss && (d_stats || d_dlogits), "ag_topk_distill: no rows or a null pointer");
    AG_REQUIRE(!d_dlogits || ldd >= V, "ag_topk_distill: gradient row stride %lld < %d logits", (long long)ldd, V);
    hipStream_t s = (hipStream_t)stream;
    const Distill p = {d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, (float)(1.0 / N)};
    // few rows too long for a workgroup's registers: the loss, then the gradient by several workgroups a row (one row of 262144 fp32: 45 -> 32 us)
    const bool apart = d_dlogits && d_stats && N <= AG_LOGITS_APART_ROWS && V / (dtype == AG_BF16 ? 8 : 4) > AG_LOGITS_HELD_PIECES, grad = d_dlogits && !apart;
    const auto bf = tail ? (grad ? distill<bf16_t, true, true> : distill<bf16_t, true, false>)
                         : (grad ? distill<bf16_t, false, true> : distill<bf16_t, false, false>);
    const auto f = tail ? (grad ? distill<float, true, true> : distill<float, true, false>)
                        : (grad ? distill<float, false, true> : distill<float, false, false>);
    if (int rc = (dtype == AG_BF16 ? bf : f)(d_logits, ld, N, V, temperature, p, d_row_loss, d_stats, d_dlogits, ldd, s)) return rc;
    hipLaunchKernelGGL(weighted_sum_kernel, dim3(1), dim3(1024), 0, s, d_row_loss, d_weights, p.weight0, N, d_loss);
    AG_LAUNCH_CHECK();
    if (!apart) return AG_OK;
    return gradient_of(dtype, tail)(d_logits, ld, N, V, temperature, p, d_stats, nullptr, nullptr, d_dlogits, ldd, s);
}

extern "C" int ag_topk_distill_bwd(const void* d_logits, int64_t ld, int N, int V, int dtype, float temperature, const int64_t* d_teacher_ids,
                                   const void* d_teacher_logp, int teacher_dtype, int K, const float* d_weights, int tail, const float* d_stats,
                                   const float* d_g_loss, const float* d_g_row_loss, void* d_dlogits, int64_t ldd, void* stream) {
    if (int rc = check_rows("ag_topk_distill_bwd", d_logits, ld, N, V, dtype, temperature)) return rc;
    if (int rc = check_teacher("ag_topk_distill_bwd", d_teacher_ids, d_teacher_logp, teacher_dtype, K, N)) return rc;
    AG_REQUIRE(N >= 1 && d_stats && d_dlogits, "ag_topk_distill_bwd: no rows or a null pointer");
    AG_REQUIRE(ldd >= V, "ag_topk_distill_bwd: gradient row stride %lld < %d logits", (long long)ldd, V);
    const Distill p = {d_teacher_ids, d_teacher_logp, teacher_dtype, K, d_weights, (float)(1.0 / N)};
    return gradient_of(dtype, tail)(d_logits, ld, N, V, temperature, p, d_stats, d_g_loss, d_g_row_loss, d_dlogits, ldd, (hipStream_t)stream);
}
