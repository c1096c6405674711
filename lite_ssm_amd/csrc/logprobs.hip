// logprobs.hip — log probabilities of given tokens under rows of logits, their
// entropies and best alternatives, and the gradient to the logits.
//
// A row x of V logits and a token t:
//   m = max x,  S = sum e^{x - m},  ls = log S,  T = sum e^{x - m} (x - m)
//   log p(v) = (x_v - m) - ls,  H = -sum p log p = ls - T / S
//   d log p(t) / dx_v = [v = t] - p_v,  dH / dx_v = -p_v (log p_v + H)
// (max, ls) are kept instead of log-sum-exp: their sum would lose up to
// 2^-24 |m| where the two numbers do not.
//
// A block reads one segment of a row into registers, once: all of its loads
// are in flight together, and the maximum, the sums, the alternatives and the
// gradient are passes over registers.  A row that does not fit one block's
// registers, or one of few rows, is cut into segments that a second launch
// joins.  Bound: the logits' bytes (8000 x 50280 bf16: 182 us, 4.4 TB/s; with the
// gradient 2048 x 50280: 94 us, 4.4 TB/s read and written); with few rows the
// latency of the load, the passes and the launches.
//
// Masked logits: -inf has p = 0 and adds nothing (p log p is 0 there);
// the type's lowest value is an ordinary number.  A row with nothing but -inf
// has log p = -inf, H = 0, statistics (0, inf) and a zero gradient.  A NaN or
// +inf makes its row NaN.
#include <algorithm>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "internal.hpp"

namespace lssm {

namespace {

constexpr uint32_t LP_MAXR = 8;              // 16-byte vectors a thread holds
constexpr uint32_t LP_WIDE = 1024, LP_SMALL = 256;   // threads of a segment's block
constexpr int LP_CAP = 1024;                 // candidates of a segment's alternatives
constexpr uint32_t LP_MAXS = 128;             // segments of a row
constexpr int LP_JOIN = LSSM_LOGPROB_MAX_TOP * (LSSM_LOGPROB_MAX_TOP + 1) / 2;
static_assert(LSSM_LOGPROB_MAX_VOCAB / 4 <= LP_MAXS * LP_WIDE * LP_MAXR, "segments");
static_assert(LP_JOIN % 8 == 0 && LP_CAP % 8 == 0, "lists");
constexpr float LOG2E = 1.44269504088896341f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

__device__ __forceinline__ float mul0(float a, float b) { return a == 0.0f ? 0.0f : a * b; }
__device__ __forceinline__ float exp_fast(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
// An exponent as a factor of its own e^d: below -200 e^d is 0, and so is the
// product, also for -inf.  (A NaN is lost here; e^d keeps it.)
__device__ __forceinline__ float factor(float d) { return fmaxf(d, -200.0f); }

template <typename T> struct Vec { static constexpr int E = 16 / sizeof(T); };

// element e (compile-time after unrolling) of a 16-byte vector
template <typename T> __device__ __forceinline__ float elem(const u32x4& q, int e) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(q[e]);
    } else {
        const uint32_t w = q[e / 2];
        if constexpr (__is_same(T, bf16)) return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
        else return f_of_bits<T>((uint16_t)((e & 1) ? (w >> 16) : w));
    }
}
template <typename T> __device__ __forceinline__ uint32_t neg_inf_word() {
    return sizeof(T) == 4 ? 0xff800000u : (__is_same(T, bf16) ? 0xff80ff80u : 0xfc00fc00u);
}

// Order of the alternatives: larger value first, then the lower index.  0: no
// alternative (-inf, NaN).  -0 and +0 are equal.
__device__ __forceinline__ uint32_t ord_of(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_ord(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ u64 key_of(uint32_t ord, uint32_t idx) { return ((u64)ord << 32) | (uint32_t)~idx; }

// Maximum over the wave, in every lane.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x141>(v));
    v = fmaxf(v, dpp_f32<0x140>(v));
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// (m, S, T) of a set of logits relative to its maximum m; moved to a larger
// reference M.  An empty set is (-FLT_MAX, 0, 0).
struct Soft { float m, S, T; };
__device__ __forceinline__ Soft moved(Soft a, float M) {
    const float d = a.m - M, f = d == 0.0f ? 1.0f : exp_fast(d);
    return {M, a.S * f, mul0(f, a.T + mul0(a.S, d))};
}

// Keeps a pass over the registers from leaving its unpacked values to the next
// (16-bit logits: twice the registers, and spills).
template <int R> __device__ __forceinline__ void repack(u32x4 (&q)[R]) {
#pragma unroll
    for (int i = 0; i < R; ++i) asm volatile("" : "+v"(q[i]));
}

// Lane 0's sums for the whole wave: a multiplication may be folded into the
// lanes' first addition, whose two sides then round differently.
__device__ __forceinline__ Soft same(Soft a) { return {a.m, readlane_f(a.S, 0), readlane_f(a.T, 0)}; }

// What a row gives in the end.
struct RowOut { float max, ls, H; };
__device__ __forceinline__ RowOut row_out(Soft a) {
    if (a.S == 0.0f) return {0.0f, INFINITY, 0.0f};     // nothing left
    const float ls = logf(a.S);
    return {a.m < INFINITY ? a.m + 0.0f * ls : a.m, ls, ls - a.T / a.S};     // (a NaN shows in the maximum too)
}

__device__ __forceinline__ void store_row(const LogprobArgs& a, uint32_t r, const RowOut& o, float xt, int t) {
    if (a.logprob) a.logprob[r] = t < 0 ? 0.0f : ((uint32_t)t < a.V ? (xt - o.max) - o.ls : NAN);
    if (a.entropy) a.entropy[r] = o.H;
    if (a.stats) {
        a.stats[2 * (size_t)r] = o.max;
        a.stats[2 * (size_t)r + 1] = o.ls;
    }
    if (t >= 0 && (uint32_t)t >= a.V) atomicOr(a.status, STATUS_BAD_TARGET);
}

// The K best of n unique keys in LDS: the rank of a key is the number of
// larger ones, so the order in which they were collected does not show.  Four
// lanes a key, each a quarter of the others (the list is filled up with zeros
// to a multiple of 8, which are larger than none).
template <int NT, typename F> __device__ __forceinline__ void rank_keys(u64* keys, uint32_t n, uint32_t K, F put) {
    const uint32_t n8 = (n + 7) & ~7u, part = threadIdx.x % 4;
    if (n + threadIdx.x < n8) keys[n + threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < n; i0 += NT / 4) {
        const uint32_t i = i0 + threadIdx.x / 4;
        const u64 k = i < n ? keys[i] : ~0ull;
        int rank = 0;
#pragma unroll 4
        for (uint32_t j = 2 * part; j < n8; j += 8) rank += (keys[j] > k ? 1 : 0) + (keys[j + 1] > k ? 1 : 0);
        rank += __builtin_amdgcn_update_dpp(0, rank, 0xB1, 0xF, 0xF, false);
        rank += __builtin_amdgcn_update_dpp(0, rank, 0x4E, 0xF, 0xF, false);
        if (part == 0 && i < n && (uint32_t)rank < K) put((uint32_t)rank, k);
    }
}

// Gradient of one logit; p = 0 where it is masked, whatever log p is.
__device__ __forceinline__ float grad_of(float x, float max, float ls, float H, float g, float ge) {
    const float lp = (x - max) - ls, p = exp_fast(lp);
    return -p * fmaf(ge, factor(lp) + H, g);
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, from_f<T>(a)) |
           ((uint32_t)__builtin_bit_cast(uint16_t, from_f<T>(b)) << 16);
}

// Where a row's 16-byte vectors lie: `head` elements before the first aligned
// address, then nv vectors, the rest behind them.
template <typename T> struct RowSpan {
    uint32_t head, nv, tail0;
    __device__ RowSpan(const T* row, uint32_t V) {
        head = min(V, (uint32_t)(((16u - ((uintptr_t)row & 15u)) & 15u) / sizeof(T)));
        nv = (V - head) / Vec<T>::E;
        tail0 = head + nv * Vec<T>::E;
    }
};

// One segment of a row (the whole row where a.S == 1).  Alternatives: a value no
// less than K of the block's is found from the lanes' maxima, what lies above it
// is collected (a K or two) and ranked.  They cost 1.6 us with K = 1 and 5
// with 64 in a block of few rows (1 x 50280: 3.1 us without, 4.7 and 8.3 with), 3
// and 6 in a block of LP_WIDE threads; only more equal values than the list
// holds take further passes, over the registers.
// GRAD (a.S == 1, no alternatives): the gradient is written from the registers too.
template <typename T, int R, bool GRAD, int LP_NT>
__global__ __launch_bounds__(LP_NT, 8) void logprob_seg_kernel(LogprobArgs a) {
    constexpr int E = Vec<T>::E, LP_NW = LP_NT / WAVE;
    constexpr int LP_TAIL = LP_NT / 2;       // first thread of those that take a row's ragged end
    __shared__ float sm[LP_NW], sS[LP_NW], sT[LP_NW];
    __shared__ uint32_t stau[LP_NW], stau2[LP_NW], scount;
    __shared__ u64 keys[LP_CAP];
    __shared__ u64 swin[LP_NW];
    const uint32_t r = blockIdx.x / a.S, seg = blockIdx.x % a.S;
    const uint32_t tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const T* row = (const T*)a.x + (size_t)r * a.stride;
    const RowSpan<T> sp(row, a.V);
    const uint32_t v0 = seg * a.seg_vecs, v1 = min(sp.nv, v0 + a.seg_vecs);
    const u32x4* vecs = reinterpret_cast<const u32x4*>(row + sp.head);

    u32x4 q[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint32_t v = v0 + i * LP_NT + tid;
        const uint32_t n = neg_inf_word<T>();
        q[i] = v < v1 ? vecs[v] : u32x4{n, n, n, n};
    }
    // the ragged ends: threads 0.. those before the first vector (first
    // segment), threads LP_TAIL.. those behind the last (last segment)
    float xe = -INFINITY;
    uint32_t ie = a.V;
    if (seg == 0 && tid < sp.head) ie = tid;
    if (seg + 1 == a.S && tid >= LP_TAIL && sp.tail0 + (tid - LP_TAIL) < a.V) ie = sp.tail0 + (tid - LP_TAIL);
    if (ie < a.V) xe = to_f(row[ie]);

    // the given token's logit, read before any gradient may replace it
    int t = -1;
    float xt = 0.0f;
    if ((GRAD || tid == 0) && a.S == 1 && a.tokens) {
        t = a.tokens[r];
        if (tid == 0 && t >= 0 && (uint32_t)t < a.V) xt = to_f(row[t]);
    }

    float m = fmaxf(-FLT_MAX, xe);
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, elem<T>(q[i], e));
        __builtin_amdgcn_sched_barrier(0);
    }
    repack(q);
    float S, U;
    {
        const float d = xe - m;
        S = exp_fast(d);
        U = S * factor(d);
    }
    float S2 = 0.0f, U2 = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = elem<T>(q[i], e) - m, x = exp_fast(d);
            (e & 1 ? S2 : S) += x;
            (e & 1 ? U2 : U) = fmaf(x, factor(d), e & 1 ? U2 : U);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    S += S2;
    U += U2;
    const float mw = wave_max(m);
    Soft s = moved({m, S, U}, mw);
    s.S = wave_sum(s.S);
    s.T = wave_sum(s.T);
    const uint32_t K = GRAD ? 0u : a.K;
    if (tid % WAVE == 0) {
        sm[w] = mw;
        sS[w] = s.S;
        sT[w] = s.T;
    }
    if (K) {
        // Two values that at least K of the block's are no less than: the K-th
        // best of a wave's lanes' best values, and the lowest of the waves'
        // ceil(K / waves)-th best ones.  Either may be the larger.  Found bit
        // by bit, down to the last that a 16-bit logit has, or to 2^-13 of fp32's
        // (lower ones would only shorten the list).
        constexpr int last = sizeof(T) == 4 ? 10 : (__is_same(T, bf16) ? 16 : 13);
        constexpr uint32_t nw = LP_NW;
        const uint32_t best = ord_of(m), K2 = (K + nw - 1) / nw;
        uint32_t tau = 0, tau2 = 0;
        for (int bit = 31; bit >= last; --bit) {
            const uint32_t c = tau | (1u << bit), c2 = tau2 | (1u << bit);
            if ((uint32_t)__popcll(__ballot(best >= c)) >= K) tau = c;
            if ((uint32_t)__popcll(__ballot(best >= c2)) >= K2) tau2 = c2;
        }
        if (tid % WAVE == 0) {
            stau[w] = tau;
            stau2[w] = tau2;
        }
        if (tid == 0) scount = 0;
    }
    __syncthreads();
    // all waves' sums (lanes 16 and up repeat the first 16)
    const int l = tid % LP_NW;
    const float M = wave_max(sm[l]);
    Soft b = moved({sm[l], sS[l], sT[l]}, M);
    b.S = group_sum<LP_NW>(b.S);
    b.T = group_sum<LP_NW>(b.T);
    b = same(b);
    const RowOut o = row_out(b);
    if (tid == 0) {
        if (a.S == 1) {
            store_row(a, r, o, xt, t);
        } else {
            float* p = a.part + 3 * (size_t)blockIdx.x;
            p[0] = b.m;
            p[1] = b.S;
            p[2] = b.T;
        }
    }
    if (K) {
        uint32_t tau = ord_of(-FLT_MAX), tau2 = ~0u;
#pragma unroll 4
        for (int i = 0; i < LP_NW; ++i) {
            tau = max(tau, stau[i]);
            tau2 = min(tau2, stau2[i]);
        }
        tau = max(tau, tau2);
        const float least = of_ord(tau);
        auto each = [&](auto f) {
            repack(q);
            uint32_t vb = v0 + tid;
            asm volatile("" : "+v"(vb));       // nor its places
            if (ie < a.V) f(xe, ie);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t v = vb + i * LP_NT;
                if (v < v1) {
#pragma unroll
                    for (int e = 0; e < E; ++e) f(elem<T>(q[i], e), sp.head + v * E + e);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (m >= least)
            each([&](float v, uint32_t idx) {
                if (v >= least) {
                    const uint32_t at = atomicAdd(&scount, 1u);
                    if (at < LP_CAP) keys[at] = key_of(ord_of(v), idx);
                }
            });
        __syncthreads();
        const uint32_t n = scount;
        auto put = [&](uint32_t rank, u64 k) {
            const uint32_t idx = ~(uint32_t)k;
            if (a.S == 1) {
                const float v = of_ord((uint32_t)(k >> 32));
                a.top_ids[(size_t)r * K + rank] = k ? (int)idx : -1;
                a.top_logprobs[(size_t)r * K + rank] = k ? (v - o.max) - o.ls : -INFINITY;
            } else {
                a.part_keys[(size_t)blockIdx.x * K + rank] = k;
            }
        };
        if (n <= LP_CAP) {
            rank_keys<LP_NT>(keys, n, K, put);
            for (uint32_t i = n + tid; i < K; i += LP_NT) put(i, 0);
        } else {
            // more equal (or masked) values than the list holds: one after the
            // other, the best key below the last
            u64 last = ~0ull;
            for (uint32_t i = 0; i < K; ++i) {
                u64 k = 0;
                each([&](float v, uint32_t idx) {
                    const uint32_t ov = ord_of(v);
                    const u64 c = ov ? key_of(ov, idx) : 0;
                    if (c < last && c > k) k = c;
                });
#pragma unroll
                for (int sft = 1; sft < WAVE; sft <<= 1) {
                    const u64 c = __shfl_xor(k, sft);
                    k = c > k ? c : k;
                }
                if (tid % WAVE == 0) swin[w] = k;
                __syncthreads();
                k = 0;
                for (int j = 0; j < LP_NW; ++j) k = swin[j] > k ? swin[j] : k;
                __syncthreads();
                if (tid == 0) put(i, k);
                last = k;
            }
        }
    }
    if constexpr (GRAD) {
        const float g = (a.g_logprob && t >= 0 && (uint32_t)t < a.V) ? a.g_logprob[r] : 0.0f;
        const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
        const float hot = o.ls == INFINITY ? 0.0f : g;
        T* dx = (T*)a.dx + (size_t)r * a.dx_stride;
        const bool vec = (((uintptr_t)dx - (uintptr_t)row) & 15u) == 0;
        repack(q);
        if (ie < a.V) dx[ie] = from_f<T>(grad_of(xe, o.max, o.ls, o.H, g, ge) + ((int)ie == t ? hot : 0.0f));
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint32_t v = v0 + i * LP_NT + tid;
            if (v < v1) {
                const uint32_t idx = sp.head + v * E;
                float d[E];
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] = grad_of(elem<T>(q[i], e), o.max, o.ls, o.H, g, ge);
                if ((uint32_t)t - idx < (uint32_t)E) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (idx + e == (uint32_t)t) d[e] += hot;
                }
                if (vec) {
                    u32x4 s4;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if constexpr (sizeof(T) == 4) s4[k] = __float_as_uint(d[k]);
                        else s4[k] = pack2<T>(d[2 * k], d[2 * k + 1]);
                    }
                    *reinterpret_cast<u32x4*>(dx + idx) = s4;
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) dx[idx + e] = from_f<T>(d[e]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Joins a row's segments: the sums, then the best of the segments' best.  A
// block a row, one wave for the sums; latency only (2.4 us without alternatives,
// 4 to 5 with 20).
template <typename T> __global__ __launch_bounds__(256) void logprob_join_kernel(LogprobArgs a) {
    const uint32_t r = blockIdx.x, tid = threadIdx.x, S = a.S, K = a.K;
    // all first loads at once
    const u64* in = a.part_keys + (size_t)r * S * K;
    const u64 mine = tid < S * K ? in[tid] : 0;
    u64 head = 0, late = 0;
    if (K && tid < S) {
        head = in[(size_t)tid * K];
        late = in[(size_t)tid * K + (K + S - 1) / S - 1];
    }
    int t = -1;
    float xt = 0.0f;
    if (tid == 0 && a.tokens) {
        t = a.tokens[r];
        if (t >= 0 && (uint32_t)t < a.V) xt = to_f(((const T*)a.x)[(size_t)r * a.stride + t]);
    }
    const float* p = a.part + 3 * (size_t)r * S;
    Soft s{-FLT_MAX, 0.0f, 0.0f};
    for (uint32_t i = tid % WAVE; i < S; i += WAVE) {
        const Soft n{p[3 * i], p[3 * i + 1], p[3 * i + 2]};
        const float M = fmaxf(s.m, n.m);
        const Soft x = moved(s, M), y = moved(n, M);
        s = {M, x.S + y.S, x.T + y.T};
    }
    s = moved(s, wave_max(s.m));
    s.S = wave_sum(s.S);
    s.T = wave_sum(s.T);
    s = same(s);
    const RowOut o = row_out(s);
    if (tid == 0) store_row(a, r, o, xt, t);
    if (K == 0) return;
    // A segment's keys are in order: the i-th of the segment whose best has
    // rank h among the segments' is behind i of its own and h others, so only
    // those with h + i < K are looked at, K (K + 1) / 2 at most; and none
    // below the lowest of all segments' ceil(K / S)-th keys.
    __shared__ u64 keys[LP_JOIN];
    __shared__ uint32_t rank[LP_MAXS], count, found;
    if (tid < S) {
        keys[tid] = head;
        keys[LP_MAXS + tid] = late;
    }
    if (tid == 0) count = found = 0;
    __syncthreads();
    if (tid < S) {
        uint32_t h = 0;
        for (uint32_t j = 0; j < S; ++j) h += keys[j] > head ? 1u : 0u;
        rank[tid] = h;
    }
    u64 least = ~0ull;
    for (uint32_t j = 0; j < S; ++j) least = min(least, keys[LP_MAXS + j]);
    __syncthreads();
    for (uint32_t i = tid; i < S * K; i += 256) {
        const uint32_t sg = i / K;
        if (rank[sg] + (i - sg * K) < K) {
            const u64 k = i == tid ? mine : in[i];
            if (k && k >= least) keys[atomicAdd(&count, 1u)] = k;      // 0: an empty place
        }
    }
    __syncthreads();
    rank_keys<256>(keys, count, K, [&](uint32_t place, u64 k) {
        atomicAdd(&found, 1u);
        a.top_ids[(size_t)r * K + place] = (int)~(uint32_t)k;
        a.top_logprobs[(size_t)r * K + place] = (of_ord((uint32_t)(k >> 32)) - o.max) - o.ls;
    });
    __syncthreads();
    for (uint32_t i = found + tid; i < K; i += 256) {
        a.top_ids[(size_t)r * K + i] = -1;
        a.top_logprobs[(size_t)r * K + i] = -INFINITY;
    }
}

// The gradient from kept statistics: one pass, a block a stretch of a row of
// LG_R vectors a thread, a read and a write of 16 bytes apiece; bound by them
// (700 x 256000 bf16: 121 us, 5.9 TB/s with the logits partly in the last-level
// cache; splitting the rows so that more of them stay there measured no faster:
// 217 us for loss and gradient at once, 226 in two, 275 in five).
constexpr int LG_NT = 256, LG_R = 4;
template <typename T> __global__ __launch_bounds__(LG_NT) void logprob_grad_kernel(LogprobArgs a) {
    constexpr int E = Vec<T>::E;
    const uint32_t r = blockIdx.x / a.S, seg = blockIdx.x % a.S, tid = threadIdx.x;
    const T* row = (const T*)a.x + (size_t)r * a.stride;
    T* dx = (T*)a.dx + (size_t)r * a.dx_stride;
    const RowSpan<T> sp(row, a.V);
    const u32x4* vecs = reinterpret_cast<const u32x4*>(row + sp.head);
    const uint32_t v0 = seg * (LG_NT * LG_R);
    u32x4 q[LG_R];
#pragma unroll
    for (int i = 0; i < LG_R; ++i) {
        const uint32_t v = v0 + i * LG_NT + tid;
        q[i] = v < sp.nv ? vecs[v] : u32x4{0, 0, 0, 0};
    }
    const float mx = a.stats[2 * (size_t)r], ls = a.stats[2 * (size_t)r + 1];
    const float H = a.entropy ? a.entropy[r] : 0.0f;
    const int t = a.tokens ? a.tokens[r] : -1;
    const float g = (a.g_logprob && t >= 0 && (uint32_t)t < a.V) ? a.g_logprob[r] : 0.0f;
    const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
    const float hot = ls == INFINITY ? 0.0f : g;
    if (seg == 0 && tid == 0 && t >= 0 && (uint32_t)t >= a.V) atomicOr(a.status, STATUS_BAD_TARGET);
    const bool vec = (((uintptr_t)dx - (uintptr_t)row) & 15u) == 0;
    uint32_t ie = a.V;
    if (seg == 0 && tid < sp.head) ie = tid;
    if (seg == 0 && tid >= LG_NT / 2 && sp.tail0 + (tid - LG_NT / 2) < a.V) ie = sp.tail0 + (tid - LG_NT / 2);
    if (ie < a.V) dx[ie] = from_f<T>(grad_of(to_f(row[ie]), mx, ls, H, g, ge) + ((int)ie == t ? hot : 0.0f));
#pragma unroll
    for (int i = 0; i < LG_R; ++i) {
        const uint32_t v = v0 + i * LG_NT + tid;
        if (v >= sp.nv) continue;
        const uint32_t idx = sp.head + v * E;
        float d[E];
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = grad_of(elem<T>(q[i], e), mx, ls, H, g, ge);
        if ((uint32_t)t - idx < (uint32_t)E) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (idx + e == (uint32_t)t) d[e] += hot;
        }
        if (vec) {
            u32x4 s4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) s4[k] = __float_as_uint(d[k]);
                else s4[k] = pack2<T>(d[2 * k], d[2 * k + 1]);
            }
            *reinterpret_cast<u32x4*>(dx + idx) = s4;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) dx[idx + e] = from_f<T>(d[e]);
        }
    }
}

template <typename F> hipError_t with_type(int act, F f) {
    if (act == LSSM_BF16) return f(bf16{});
    if (act == LSSM_F16) return f(f16{});
    return f(float{});
}

}  // namespace

// How a row is cut: segments, threads a block, 16-byte vectors a thread (the
// least that hold a segment: 4096 rows of 8000 take 36 us so, 79 at 8).
//   - A row that LP_SMALL threads hold is one segment of theirs: 4096 rows, bf16,
//     of LP_WIDE -> of LP_SMALL threads: 2000 logits 33.6 -> 10.6 us, 8000 35.1
//     -> 18.3, 16000 37.1 -> 28.5 (loss and gradient 61.1 -> 55.3).
//   - A longer one is cut for LP_WIDE threads, a segment as long as LP_MAXR
//     vectors allow: 2048 x 50280 in one pass of 93.8 us with its gradient, cut
//     in two (LP_MAXR 4) 130; 8000 x 50280 with 5 alternatives 215 and 294.
//   - Where all this makes fewer than LP_FEW blocks, it is cut finer, for
//     LP_SMALL threads, as far as LP_WANT blocks go: 1 x 50280 with 5
//     alternatives 11.5 -> 9.3, 8 rows of those 12.4 -> 9.8, 1 x 256000 with 20
//     16.6 -> 14.8; 32 x 50280 with 20 12.4 both, 64 without any 7.2 -> 8.4, 128
//     with 5 11.9 -> 14.3.  (LP_WANT 256 and 1024 measured alike.)
//   - Rows of several segments that make LP_HALF blocks at most, half the CUs,
//     are cut in twice as many: 10 x 256000 with 20 alternatives 16.6 -> 14.0, 32 of
//     those 17.4 -> 15.6; 50 of them 18.2 -> 19.9.
constexpr uint32_t LP_FEW = 32, LP_HALF = 128, LP_WANT = 512;
struct LogprobPlan { uint32_t S, nt, R; };
static LogprobPlan plan_of(uint32_t rows, uint32_t vocab, int act) {
    const uint32_t nv = std::max(1u, vocab / (act == LSSM_F32 ? 4u : 8u));
    auto segs = [&](uint32_t nt, uint32_t R) { return (nv + nt * R - 1) / (nt * R); };
    const uint32_t S = segs(LP_WIDE, LP_MAXR);
    uint32_t R = 2;
    if ((uint64_t)rows * S < LP_FEW && segs(LP_SMALL, LP_MAXR) <= LP_MAXS) {
        while (R < LP_MAXR && (rows * segs(LP_SMALL, R) > LP_WANT || segs(LP_SMALL, R) > LP_MAXS)) R *= 2;
        return {segs(LP_SMALL, R), LP_SMALL, R};
    }
    const uint32_t nt = nv <= LP_SMALL * LP_MAXR ? LP_SMALL : LP_WIDE;
    if (S > 1 && (uint64_t)rows * S <= LP_HALF) return {segs(LP_WIDE, LP_MAXR / 2), LP_WIDE, LP_MAXR / 2};
    while (R < LP_MAXR && segs(nt, R) > S) R *= 2;
    return {S, nt, R};
}

uint32_t logprob_segments(uint32_t rows, uint32_t vocab, int act) { return plan_of(rows, vocab, act).S; }

// [part: 3 floats a segment, to a multiple of 8 bytes][keys: K a segment]
static size_t part_bytes(uint32_t rows, uint32_t segs) { return ((size_t)rows * segs * 12 + 7) / 8 * 8; }

// (of either type size, and enough for fewer rows too, which are cut finer)
size_t logprob_ws_bytes(uint32_t rows, uint32_t vocab, uint32_t top_k) {
    size_t n = 0;
    auto of = [&](uint32_t r) {
        for (int act : {LSSM_BF16, LSSM_F32}) {
            const uint32_t S = plan_of(r, vocab, act).S;
            if (S > 1) n = std::max(n, part_bytes(r, S) + (size_t)r * S * top_k * 8);
        }
    };
    for (uint32_t r = 1; r < std::min(rows, LP_HALF + 1); ++r) of(r);
    of(rows);
    return n;
}

hipError_t launch_logprobs(hipStream_t s, LogprobArgs a, int act, void* ws) {
    const LogprobPlan p = plan_of(a.rows, a.V, act);
    const uint32_t nv = std::max(1u, a.V / (act == LSSM_F32 ? 4u : 8u));
    a.S = p.S;
    a.seg_vecs = (nv + p.S - 1) / p.S;
    if (a.S > 1) {
        a.part = static_cast<float*>(ws);
        a.part_keys = reinterpret_cast<unsigned long long*>(static_cast<char*>(ws) + part_bytes(a.rows, a.S));
    }
    return with_type(act, [&](auto z) {
        using T = decltype(z);
        const dim3 grid(a.rows * a.S);
        const bool grad = a.dx && a.S == 1;
        auto go = [&](auto rc, auto ntc) {
            constexpr int R = decltype(rc)::value, NT = decltype(ntc)::value;
            if (grad) logprob_seg_kernel<T, R, true, NT><<<grid, NT, 0, s>>>(a);
            else logprob_seg_kernel<T, R, false, NT><<<grid, NT, 0, s>>>(a);
        };
        constexpr std::integral_constant<int, LP_SMALL> small;
        constexpr std::integral_constant<int, LP_WIDE> wide;      // (rows of more than LP_SMALL 8 vectors: R 4 or 8)
        if (p.nt == LP_SMALL) {
            if (p.R == 2) go(std::integral_constant<int, 2>{}, small);
            else if (p.R == 4) go(std::integral_constant<int, 4>{}, small);
            else go(std::integral_constant<int, 8>{}, small);
        } else {
            if (p.R <= 4) go(std::integral_constant<int, 4>{}, wide);
            else go(std::integral_constant<int, 8>{}, wide);
        }
        if (a.S > 1) logprob_join_kernel<T><<<a.rows, 256, 0, s>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !a.dx || grad) return e;
        return launch_logprobs_grad(s, a, act);
    });
}

hipError_t launch_logprobs_grad(hipStream_t s, LogprobArgs a, int act) {
    const uint32_t nv = a.V / (act == LSSM_F32 ? 4u : 8u);
    a.S = std::max(1u, (nv + LG_NT * LG_R - 1) / (LG_NT * LG_R));
    return with_type(act, [&](auto z) {
        logprob_grad_kernel<decltype(z)><<<a.rows * a.S, LG_NT, 0, s>>>(a);
        return hipGetLastError();
    });
}

}  // namespace lssm
