// ssd_bwd.hip — gradients of the SSD scan (lssm_ssd_chunked).
//
// Forward, a head with state h [P, N], dt_t = clamp(softplus(raw_t + bias)), A = -e^A_log:
//   h_t = e^{A dt_t} h_{t-1} + dt_t x_t B_t^T,   y_t = h_t C_t + D x_t
// Backward, G_t = dL / dh_t (G behind the last token: the given d_state):
//   G_t = dy_t C_t^T + e^{A dt_{t+1}} G_{t+1}
//   dC_t = sum_heads h_t^T dy_t,   dB_t = sum_heads dt_t G_t^T x_t
//   dx_t = dt_t G_t B_t + D dy_t,  dD = sum dy_t.x_t
//   a_t = e^{A dt_t} <G_t, h_{t-1}>,  ddt_t = x_t.(G_t B_t) + A a_t,  dA = sum dt_t a_t
//
// In chunks, with Lc the inclusive sum of A dt from the chunk's start, Lq its
// last value, h0 the state that enters the chunk and G1 the gradient of the one
// that leaves it, and E[t, j] = e^{Lc_t - Lc_j} (j <= t):
//   S[t, j] = (dy_t.x_j) E,  M[t, j] = (C_t.B_j) E
//   dC_t  = e^{Lc_t} h0^T dy_t + sum_j S[t, j] dt_j B_j
//   dB_j  = dt_j (e^{Lq - Lc_j} G1^T x_j + sum_t S[t, j] C_t)
//   dx'_j = e^{Lq - Lc_j} G1 B_j + sum_t M[t, j] dy_t,  dx_j = dt_j dx'_j + D dy_j
// The within-chunk parts of dB and dC need sum_heads S only: the heads of a
// group share B and C.  a_t is the sum over all pairs of a source before t and
// a sink from t on,
//   a_t = e^{Lq} <G1, h0> + sum_{j < t} u_j + sum_{s >= t} v_s
//         + sum_{s >= t > j} K[s, j],
//   u_j = dt_j e^{Lq - Lc_j} x_j.(G1 B_j),  v_s = e^{Lc_s} C_s.(h0^T dy_s),
//   K[s, j] = (dy_s.x_j)(C_s.B_j) E dt_j
// which adds terms of one chunk only, and only terms that the step's own decay is
// part of: none is formed as a difference of longer sums, so a step that forgets
// what came before it (A dt far below 0) keeps its gradient's digits.
//
// Three steps: the states h0 (forwards) and G1 (backwards) of every chunk are
// kept; the chunks' gradients, in parallel; sums over heads, slices and chunks.
// Every order of summation is fixed.
//
// Two forms.  The bf16 one (second half of this file) takes bf16 with N = 128, P
// in 64s and 16-byte aligned arrays, the generic one everything else.  Us,
// generic -> bf16 form, same inputs: a 130M layer (24 heads) of 37 tokens 34.1 ->
// 34.6, 128 40.0 -> 35.8, 512 62.8 -> 47.0, 2048 150 -> 76; a 2.7B layer (80 heads)
// of 37 tokens 61 -> 44, 4096 951 -> 241, 4 x 4096 3842 -> 722.  (At one token of 24
// heads the generic form is 3 us faster; no rule is made for that.)
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.hpp"
#include "internal.hpp"

namespace lssm {

namespace {

__device__ __forceinline__ floatx4 mma4(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Any type, head size and state size (N <= 256), fp32 products
// (v_mfma_f32_16x16x4_f32): chunks of 32 tokens, slices of 32 state rows.
// Every chunk's own state in parallel, then the scan over the chunks, in place.
// The sums of A dt are held in 64 bits: differences of sums that grow along a
// chunk are what every decay is the exponential of.
// ---------------------------------------------------------------------------
// A step's A dt below this is taken as this: e^-104 is 0 in fp32 and so is every
// decay over such a step, and the sums behind it stay small enough to hold the
// steps that follow.  (A NaN stays one.)
constexpr double LEAST_STEP = -104.0;
__device__ __forceinline__ double bounded(double x) { return x < LEAST_STEP ? LEAST_STEP : x; }

constexpr int GQ = 32;      // tokens a chunk
constexpr int GP = 32;      // state rows a slice
constexpr int GXP = 36;     // LDS pitch of a [token][row] tile (= 4 modulo 64 banks x 9)
constexpr int G_NT = 256;

// slope of dt in v = raw + bias: that of the softplus sp, 0 where the clamp holds
__device__ __forceinline__ float slope_of(const SsdBwdArgs& a, float v, float sp) {
    return sp >= a.dt_min && sp <= a.dt_max ? 1.0f / (1.0f + expf(-v)) : 0.0f;
}
template <typename T> __device__ __forceinline__ float dt_slope(const SsdBwdArgs& a, uint32_t b, uint32_t t, uint32_t h) {
    const float v = to_f(((const T*)a.dt)[((size_t)b * a.L + t) * a.H + h]) + to_f(((const T*)a.dt_bias)[h]);
    return slope_of(a, v, v > 20.0f ? v : log1pf(expf(v)));
}

struct Steps { double lc, tot; float dt; };

// dt and the sums of A dt of a chunk of GQ tokens, lane t of a wave (lanes
// past GQ repeat the last token's).
template <typename T> __device__ __forceinline__ Steps chunk_steps(const SsdBwdArgs& a, uint32_t b, uint32_t h, uint32_t t0,
                                                                   uint32_t tl) {
    const uint32_t t = threadIdx.x % WAVE;
    const float A = -expf(to_f(((const T*)a.A_log)[h]));
    float dt = 0.0f;
    if (t < tl) {
        const float v = to_f(((const T*)a.dt)[((size_t)b * a.L + t0 + t) * a.H + h]) + to_f(((const T*)a.dt_bias)[h]);
        dt = v > 20.0f ? v : log1pf(expf(v));
        dt = fminf(fmaxf(dt, a.dt_min), a.dt_max);
    }
    double s = bounded((double)A * (double)dt);
#pragma unroll
    for (int d = 1; d < GQ; d <<= 1) {
        const double o = __shfl_up(s, d);
        if ((int)t >= d) s += o;
    }
    return {s, __shfl(s, GQ - 1), dt};
}

// The sums of a 16 x 16 tile's columns from each row on (the tile as its
// product leaves it: rows 4 q .. 4 q + 3 of column i), `carry` behind its last
// row; carry becomes the sum of all.
__device__ __forceinline__ void from_row(floatx4& v, float& carry) {
    v[2] += v[3];
    v[1] += v[2];
    v[0] += v[1];
    const uint32_t q = threadIdx.x / 16 % 4;
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[0]), false, false);
    const float odd = __uint_as_float(p[1]), both = __uint_as_float(p[0]) + odd;
    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(both), __float_as_uint(both), false, false);
    const float high = __uint_as_float(o[1]);
    const float after = carry + ((q % 2 ? 0.0f : odd) + (q < 2 ? high : 0.0f));
    carry += __uint_as_float(o[0]) + high;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += after;
}

// whether rows of n elements `stride` apart can be taken 16 bytes at a time
template <typename T> __device__ __forceinline__ bool whole16(const T* src, size_t stride, uint32_t n) {
    return n % (16 / sizeof(T)) == 0 && (((uintptr_t)src | (stride * sizeof(T))) & 15) == 0;
}

// A [rows <= GQ][n <= W] piece of an array of rows `stride` apart on its way
// into LDS [GQ][pitch] as fp32, zeros behind the ends, by NTH threads: get()
// loads 16 bytes at a time into registers, put() stores them.
template <typename T, int W, int NTH> struct Tile {
    static constexpr int E = 16 / sizeof(T), PER = W / E, ALL = GQ * PER, V = (ALL + NTH - 1) / NTH;
    typedef T TE __attribute__((ext_vector_type(E)));
    TE v[V];
    __device__ __forceinline__ void get(uint32_t tid, const T* src, size_t stride, uint32_t rows, uint32_t n) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t i = tid + k * NTH, r = i / PER, c = i % PER * E;
            v[k] = TE(0);
            if (r < rows && c < n) v[k] = *reinterpret_cast<const TE*>(src + r * stride + c);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = TE(0);
    }
    __device__ __forceinline__ void put(uint32_t tid, float* dst, int pitch) const {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t i = tid + k * NTH, r = i / PER, c = i % PER * E;
            if (ALL % NTH && i >= ALL) break;
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<floatx4*>(dst + r * pitch + c + e) =
                    floatx4{to_f(v[k][e]), to_f(v[k][e + 1]), to_f(v[k][e + 2]), to_f(v[k][e + 3])};
        }
    }
};
template <typename T, int W, int NTH> __device__ __forceinline__ void load_tile(float* dst, int pitch, const T* src,
                                                                                size_t stride, uint32_t rows, uint32_t n) {
    if (whole16(src, stride, n)) {
        Tile<T, W, NTH> t;
        t.get(threadIdx.x, src, stride, rows, n);
        t.put(threadIdx.x, dst, pitch);
        return;
    }
    for (uint32_t i = threadIdx.x; i < GQ * W; i += NTH) {
        const uint32_t r = i / W, c = i % W;
        dst[r * pitch + c] = (r < rows && c < n) ? to_f(src[r * stride + c]) : 0.0f;
    }
}

// What a chunk alone adds to the state behind it (direction 0: weighted outer
// products of x with B) or to the gradient in front of it (1: of dy with C):
// block (head, slice and direction; chunk; sequence).  Bound by the states it
// writes; 512 tokens of 24 heads in fp32: 13 us.  (With a walk over the chunks
// instead of this and the scan, states in registers, all launches took 232 us
// there, and 88 so.)
template <typename T, int NT> __global__ __launch_bounds__(G_NT) void ssd_bwd_own_kernel(SsdBwdArgs a) {
    constexpr int NP = NT + 4, TN = NT / 64;
    __shared__ __attribute__((aligned(16))) float Rs[GQ * GXP], Cs[GQ * NP], W[GQ];
    const uint32_t c = blockIdx.y, h = blockIdx.x / 2 / a.nslice, sl = blockIdx.x / 2 % a.nslice, p0 = sl * GP;
    const uint32_t b = blockIdx.z;
    const bool back = blockIdx.x % 2 != 0;
    const uint32_t P = a.P, N = a.N, L = a.L, pn = min((uint32_t)GP, P - p0), t0 = c * GQ, tl = min((uint32_t)GQ, L - t0);
    const uint32_t g = h / (a.H / a.G);
    const int tid = threadIdx.x, lane = tid % WAVE, li = lane % 16, lq = lane / 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
    load_tile<T, GP, G_NT>(Rs, GXP, (const T*)(back ? a.dY : a.X) + ((size_t)b * L + t0) * a.H * P + (size_t)h * P + p0,
                     (size_t)a.H * P, tl, pn);
    load_tile<T, NT, G_NT>(Cs, NP, (const T*)(back ? a.C : a.B) + ((size_t)b * L + t0) * a.G * N + (size_t)g * N, (size_t)a.G * N, tl,
                     N);
    if (w == 0) {
        const Steps st = chunk_steps<T>(a, b, h, t0, tl);
        if (lane < GQ) W[lane] = back ? expf((float)st.lc) : st.dt * expf((float)(st.tot - st.lc));
        if (lane == 0 && !back && sl == 0) a.lc[((size_t)b * a.H + h) * a.nchunk + c] = expf((float)st.tot);
    }
    __syncthreads();
    float* own = (back ? a.gst : a.hst) + (((size_t)b * a.H + h) * a.nchunk + c) * P * N;
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const uint32_t n = 16 * (w + 4 * i) + li;
            floatx4 s{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < GQ / 4; ++k) {
                const int t = 4 * k + lq;
                s = mma4(Rs[t * GXP + 16 * pt + li] * W[t], Cs[t * NP + n], s);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t p = 16 * pt + 4 * lq + r;
                if (p < pn && n < N) own[(size_t)(p0 + p) * N + n] = s[r];
            }
        }
}

// The scan: an element of a head's state a thread.  Slot c holds what chunk c
// adds and gets the state that enters it (direction 0), or the gradient of the
// one that leaves it (1).  Slots are read SC ahead; bound by reading and writing
// them (10 us at 512 tokens of 24 heads).
constexpr int SC = 8;
__global__ __launch_bounds__(G_NT) void ssd_bwd_scan_kernel(SsdBwdArgs a) {
    const uint32_t PN = a.P * a.N, i = blockIdx.x / 2 * G_NT + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    const bool back = blockIdx.x % 2 != 0;
    if (i >= PN) return;
    const size_t bh = (size_t)b * a.H + h;
    float* slots = (back ? a.gst : a.hst) + bh * a.nchunk * PN + i;
    const float* decay = a.lc + bh * a.nchunk;
    const float* init = back ? a.d_state : a.state;
    float s = init ? init[bh * PN + i] : 0.0f;
    for (uint32_t k0 = 0; k0 < a.nchunk; k0 += SC) {
        float own[SC], d[SC];
#pragma unroll
        for (int k = 0; k < SC; ++k) {
            const uint32_t q = min(k0 + k, a.nchunk - 1), c = back ? a.nchunk - 1 - q : q;
            own[k] = slots[(size_t)c * PN];
            d[k] = decay[c];
        }
#pragma unroll
        for (int k = 0; k < SC; ++k) {
            if (k0 + k >= a.nchunk) break;
            slots[(size_t)(back ? a.nchunk - 1 - (k0 + k) : k0 + k) * PN] = s;
            s = fmaf(d[k], s, own[k]);
        }
    }
    if (back && a.d_state0) a.d_state0[bh * PN + i] = s;
}

// The chunks' gradients: block = chunk, sequence, group, share of the group's
// (head, slice) pairs.  dB and dC of the share stay in registers.  NW waves;
// waves 0 .. 3 own the four tiles of S and M (tokens T0, J0) and of dx (tokens
// T0, rows J0); eight waves split the k of dx over the state's columns.  The
// next pair's rows and states are on their way into registers meanwhile, where
// they can be taken 16 bytes at a time.  Two blocks fit a CU up to N = 128.
// Bound by latency and fp32 MFMA issue: 37 us at 512 tokens of 24 heads.  Eight
// waves with the prefetch against four without: 4096 tokens of 80 heads 1519 ->
// 1104 us, N = 200 3461 -> 1831; two blocks a CU: 1104 -> 975, 1831 -> 1430.  N <= 64
// has too few columns for eight waves.
template <typename T, int NT, int NW> __global__ __launch_bounds__(64 * NW, NT == 256 ? 2 : 4) void ssd_bwd_chunk_kernel(SsdBwdArgs a) {
    constexpr int NP = NT + 4, TN = NT / (16 * NW), NTH = 64 * NW, KG = NW / 4;
    __shared__ __attribute__((aligned(16))) float Bs[GQ * NP], Hs[GP * NP], Gs[GP * NP];
    __shared__ __attribute__((aligned(16))) float Xs[GQ * GXP], Ys[GQ * GXP], Ms[GQ * GXP];
    __shared__ floatx4 part[KG > 1 ? 4 * WAVE : 1];
    __shared__ double Lc[GQ];
    __shared__ float DT[GQ], EL[GQ], ER[GQ], SL[GQ], RS[2][GQ], CS[2][GQ], VO[NW][GQ], UO[2][GQ], red[NW][2];
    const uint32_t P = a.P, N = a.N, L = a.L, hpg = a.H / a.G;
    const uint32_t c = blockIdx.x % a.nchunk, sp = blockIdx.x / a.nchunk % a.nsplit;
    const uint32_t g = blockIdx.x / a.nchunk / a.nsplit, b = blockIdx.y;
    const uint32_t t0 = c * GQ, tl = min((uint32_t)GQ, L - t0);
    int tid = threadIdx.x, lane = tid % WAVE, li = lane % 16, lq = lane / 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE), kg = w / 4;
    const int T0 = w % 4 / 2, J0 = w % 2;

    // C B^T, and C where dC's products leave it; C is not needed between
    const T* Cg = (const T*)a.C + ((size_t)b * L + t0) * a.G * N + (size_t)g * N;
    load_tile<T, NT, NTH>(Bs, NP, (const T*)a.B + ((size_t)b * L + t0) * a.G * N + (size_t)g * N, (size_t)a.G * N, tl, N);
    load_tile<T, NT, NTH>(Hs, NP, Cg, (size_t)a.G * N, tl, N);
    __syncthreads();
    floatx4 cb{0, 0, 0, 0};
    for (int k = 0; k < NT / 4; ++k)
        cb = mma4(Hs[(16 * T0 + li) * NP + 4 * k + lq], Bs[(16 * J0 + li) * NP + 4 * k + lq], cb);
    floatx4 cr[2][TN];
    floatx4 dc[2][TN], db[2][TN], ssum{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            dc[q][i] = db[q][i] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < 4; ++r) cr[q][i][r] = Hs[(16 * q + 4 * lq + r) * NP + 16 * (w + NW * i) + li];
        }

    const uint32_t pairs = hpg * a.nslice, per = (pairs + a.nsplit - 1) / a.nsplit;
    const uint32_t v_first = sp * per, v_end = min(pairs, v_first + per);
    const size_t hp = (size_t)a.H * P;
    Tile<T, GP, NTH> tx, ty;
    Tile<float, NT, NTH> th, tg;
    // (arrays and strides: the same answer for every pair)
    const bool whole = whole16((const T*)a.X, hp, P) && whole16((const T*)a.dY, hp, P) && whole16(a.hst, N, N) && GP % (16 / sizeof(T)) == 0;
    auto at = [&](uint32_t v, uint32_t& h, uint32_t& sl, size_t& row0, size_t& slot) {
        h = g * hpg + v / a.nslice;
        sl = v % a.nslice;
        row0 = ((size_t)b * L + t0) * hp + (size_t)h * P + sl * GP;
        slot = (((size_t)b * a.H + h) * a.nchunk + c) * P * N + (size_t)sl * GP * N;
    };
    auto fetch = [&](uint32_t v) {
        uint32_t h, sl;
        size_t row0, slot;
        at(v, h, sl, row0, slot);
        const uint32_t pn = min((uint32_t)GP, P - sl * GP);
        tx.get(tid, (const T*)a.X + row0, hp, tl, pn);
        ty.get(tid, (const T*)a.dY + row0, hp, tl, pn);
        th.get(tid, a.hst + slot, N, pn, N);
        tg.get(tid, a.gst + slot, N, pn, N);
    };
    if (whole && v_first < v_end) fetch(v_first);
    for (uint32_t v = v_first; v < v_end; ++v) {
        uint32_t h, sl;
        size_t row0, slot;
        at(v, h, sl, row0, slot);
        const uint32_t p0 = sl * GP, pn = min((uint32_t)GP, P - p0);
        // (places are formed again for each pair instead of being kept)
        asm volatile("" : "+v"(tid), "+v"(lane), "+v"(li), "+v"(lq));
        __syncthreads();
        if (whole) {
            tx.put(tid, Xs, GXP);
            ty.put(tid, Ys, GXP);
            th.put(tid, Hs, NP);
            tg.put(tid, Gs, NP);
        } else {
            load_tile<T, GP, NTH>(Xs, GXP, (const T*)a.X + row0, hp, tl, pn);
            load_tile<T, GP, NTH>(Ys, GXP, (const T*)a.dY + row0, hp, tl, pn);
            load_tile<float, NT, NTH>(Hs, NP, a.hst + slot, N, pn, N);
            load_tile<float, NT, NTH>(Gs, NP, a.gst + slot, N, pn, N);
        }
        if (w == NW - 1) {
            const Steps st = chunk_steps<T>(a, b, h, t0, tl);
            if (lane < GQ) {
                Lc[lane] = st.lc;
                DT[lane] = st.dt;
                EL[lane] = expf((float)st.lc);
                ER[lane] = expf((float)(st.tot - st.lc));
                SL[lane] = lane < (int)tl ? dt_slope<T>(a, b, t0 + lane, h) : 0.0f;
            }
        }
        __syncthreads();
        if (whole) {
            if (v + 1 < v_end) {
                fetch(v + 1);
            } else {
                // (not kept over the loop for this path's sake)
                tx.clear();
                ty.clear();
                th.clear();
                tg.clear();
            }
        }
        // S and M of this wave's tile; row and column sums of K
        const int j = 16 * J0 + li;
        if (kg == 0) {
            floatx4 sd{0, 0, 0, 0};
            if (T0 >= J0)
                for (int k = 0; k < GP / 4; ++k)
                    sd = mma4(Ys[(16 * T0 + li) * GXP + 4 * k + lq], Xs[(16 * J0 + li) * GXP + 4 * k + lq], sd);
            float col = 0.0f, below = 0.0f;
            floatx4 kt;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * T0 + 4 * lq + r;
                const float e = t >= j ? expf((float)(Lc[t] - Lc[j])) : 0.0f;
                const float m = cb[r] * e, kk = sd[r] * m;
                ssum[r] += sd[r] * e * DT[j];
                Ms[t * GXP + j] = m;
                kt[r] = t > j ? kk * DT[j] : 0.0f;
                col += kk;
            }
            // sinks from t on, sources of this tile before t
            from_row(kt, below);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * T0 + 4 * lq + r;
                const float row = group_sum<16>(t > j ? kt[r] : 0.0f);
                if (li == 0) RS[J0][t] = row;
            }
            col += __shfl_xor(col, 16);
            col += __shfl_xor(col, 32);
            if (lq == 0) CS[T0][j] = col;
        }
        if (kg == KG - 1) {
            // <G1, h0> and the sum of dy.x, by the last four waves
            float gh = 0.0f, yx = 0.0f;
            const int u = tid - 256 * (KG - 1);
            for (int i = u; i < GP * NT; i += 256) gh += Hs[i / NT * NP + i % NT] * Gs[i / NT * NP + i % NT];
            for (int i = u; i < GQ * GP; i += 256) yx += Xs[i / GP * GXP + i % GP] * Ys[i / GP * GXP + i % GP];
            gh = wave_sum(gh);
            yx = wave_sum(yx);
            if (lane == 0) {
                red[w % 4][0] = gh;
                red[w % 4][1] = yx;
            }
        }
        // the parts that meet the states
        float vo[2][4] = {};
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const int n = 16 * (w + NW * i) + li;
                floatx4 x{0, 0, 0, 0}, y{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < GP / 4; ++k) {
                    x = mma4(Ys[(16 * q + li) * GXP + 4 * k + lq], Hs[(4 * k + lq) * NP + n], x);
                    y = mma4(Xs[(16 * q + li) * GXP + 4 * k + lq], Gs[(4 * k + lq) * NP + n], y);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = 16 * q + 4 * lq + r;
                    const float d = EL[t] * x[r];
                    dc[q][i][r] += d;
                    vo[q][r] += d * cr[q][i][r];
                    db[q][i][r] += DT[t] * ER[t] * y[r];
                }
            }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s = group_sum<16>(vo[q][r]);
                if (li == 0) VO[w][16 * q + 4 * lq + r] = s;
            }
        floatx4 dx{0, 0, 0, 0};
#pragma unroll 8
        for (int k = 0; k < NT / 4 / KG; ++k) {
            const int n = 4 * (k + kg * (NT / 4 / KG)) + lq;
            dx = mma4(Bs[(16 * T0 + li) * NP + n], Gs[(16 * J0 + li) * NP + n], dx);
        }
        if (KG > 1 && kg == 1) part[(w % 4) * WAVE + lane] = dx;
        __syncthreads();
        if (kg == 0) {
            if (KG > 1) dx += part[w * WAVE + lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * T0 + 4 * lq + r;
                dx[r] *= ER[t];
                const float u = group_sum<16>(dx[r] * Xs[t * GXP + 16 * J0 + li]);
                if (li == 0) UO[J0][t] = u;
            }
#pragma unroll
            for (int k = 0; k < GQ / 4; ++k)
                dx = mma4(Ms[(4 * k + lq) * GXP + 16 * T0 + li], Ys[(4 * k + lq) * GXP + 16 * J0 + li], dx);
            const float D = a.D ? to_f(((const T*)a.D)[h]) : 0.0f;
            const uint32_t p = 16 * J0 + li;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t t = 16 * T0 + 4 * lq + r;
                if (t < tl && p < pn) ((T*)a.dX)[row0 + t * hp + p] = from_f<T>(fmaf(DT[t], dx[r], D * Ys[t * GXP + p]));
            }
        }
        __syncthreads();
        // a_t: pairs of a source before t and a sink from t on
        if (w == NW - 1) {
            const int t = min(lane, GQ - 1);
            const float dt = lane < GQ ? DT[t] : 0.0f, uo = UO[0][t] + UO[1][t], cs = CS[0][t] + CS[1][t];
            // sources before t with the sinks behind the chunk, and, for t in its
            // first half, with those of the second; sinks from t on with the
            // sources before the chunk
            float pre = lane < GQ ? dt * uo : 0.0f, half = lane < 15 ? dt * CS[1][t] : 0.0f, suf = 0.0f;
            if (lane < GQ)
#pragma unroll
                for (int i = 0; i < NW; ++i) suf += VO[i][t];
#pragma unroll
            for (int d = 1; d < GQ; d <<= 1) {
                const float x = __shfl_up(pre, d), y = __shfl_down(suf, d), z = __shfl_up(half, d);
                if (lane >= d) {
                    pre += x;
                    half += z;
                }
                if (lane + d < GQ) suf += y;
            }
            pre = __shfl_up(pre, 1);
            half = __shfl_up(half, 1);
            if (lane == 0) pre = 0.0f;
            if (lane == 0 || lane >= 16) half = 0.0f;
            const float edge = EL[GQ - 1] * ((red[0][0] + red[1][0]) + (red[2][0] + red[3][0]));
            const float da = (edge + pre) + (suf + ((RS[0][t] + RS[1][t]) + half));
            const float A = -expf(to_f(((const T*)a.A_log)[h]));
            float q = 0.0f;
            if (lane < (int)tl) {
                q = (uo + cs + A * da) * SL[t];
                a.q[(((size_t)sl * a.batch + b) * a.H + h) * L + t0 + lane] = q;
            }
            const float dA = wave_sum(dt * da);
            q = wave_sum(q);
            if (lane == 0) {
                float* o = a.part + ((((size_t)b * a.H + h) * a.nslice + sl) * a.nchunk + c) * 3;
                o[0] = q;
                o[1] = A * dA;
                o[2] = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
            }
        }
    }
    // within the chunk: sum of S over the share's heads with B and C
    __syncthreads();
    load_tile<T, NT, NTH>(Hs, NP, Cg, (size_t)a.G * N, tl, N);
    if (kg == 0)
#pragma unroll
        for (int r = 0; r < 4; ++r) Ms[(16 * T0 + 4 * lq + r) * GXP + 16 * J0 + li] = ssum[r];
    __syncthreads();
    const size_t base = (size_t)sp * a.share;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const uint32_t n = 16 * (w + NW * i) + li;
            for (int k = 0; k < GQ / 4; ++k) {
                dc[q][i] = mma4(Ms[(16 * q + li) * GXP + 4 * k + lq], Bs[(4 * k + lq) * NP + n], dc[q][i]);
                db[q][i] = mma4(Ms[(4 * k + lq) * GXP + 16 * q + li], Hs[(4 * k + lq) * NP + n], db[q][i]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t t = 16 * q + 4 * lq + r;
                if (t < tl && n < N) {
                    const size_t at = base + (((size_t)b * L + t0 + t) * a.G + g) * N + n;
                    a.cpart[at] = dc[q][i][r];
                    a.bpart[at] = db[q][i][r];
                }
            }
        }
}

// ---------------------------------------------------------------------------
// bf16, N = 128, P a multiple of 64: chunks of 128 tokens, slices of 64 state
// rows, v_mfma_f32_16x16x32_bf16.  An operand formed in fp32 (weighted rows,
// states, M, the heads' sum of S) enters as a sum of bf16 pieces, each the
// rounding of what the pieces before it left: two pieces hold it to 2^-17,
// three to 2^-25.  What an operand of 16 bits holds already is exact.
// The 16x16x32 operands: lane l = 16 q + i supplies row / column i, k = 8 q ..
// 8 q + 7; the result holds rows 4 q .. 4 q + 3 of column i.  Operands whose k
// runs down the rows of a tile are read with the transposing LDS load.
// ---------------------------------------------------------------------------
constexpr int FQ = 128;      // tokens a chunk
constexpr int FP = 64;       // state rows a slice
constexpr int FN = 128;      // state size
constexpr int FXP = FP + 8;  // pitch of a [token or n][row] tile
constexpr int FBP = FN + 16; // pitch of a [token][n] tile
constexpr int F_NT = 512;

typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// LDS traffic only: global loads and stores stay in flight across it
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ floatx4 mma(s8v a, s8v b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// lane i of each 16 lanes: column i of four rows, one row of each four lanes
__device__ __forceinline__ s4v ld_tr(const bf16* p) {
    typedef __attribute__((address_space(3))) s4v lds_s4v;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v*)(const_cast<bf16*>(p)));
}
__device__ __forceinline__ s8v cat8(s4v lo, s4v hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ float val(short b) { return __uint_as_float((uint32_t)(uint16_t)b << 16); }

// a buffer of `bytes` from p on: loads past its end give 0
__device__ __forceinline__ auto rsrc(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// v rounded to bf16; v becomes what is left
__device__ __forceinline__ s4v take4(floatx4& v) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const uint32_t a = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[0], v[1]}, bf16x2));
    const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2], v[3]}, bf16x2));
    v[0] -= __uint_as_float(a << 16);
    v[1] -= __uint_as_float(a & 0xffff0000u);
    v[2] -= __uint_as_float(b << 16);
    v[3] -= __uint_as_float(b & 0xffff0000u);
    return __builtin_bit_cast(s4v, u32x2{a, b});
}

// The sums of A dt in the bf16 form: -Lc in units of 2^-18 (at most 128 104 2^18
// < 2^32).  A decay's exponent is a difference of two, exact, each rounded by
// 2^-19 whatever the sums have grown to (an fp32 sum passes that at 64); what
// they decay is written in 16 bits.  The states' weights are formed from the
// sums themselves.
constexpr float LC_UNIT = 1.0f / 262144.0f;
constexpr uint32_t LC_NAN = ~0u;
__device__ __forceinline__ uint32_t to_units(double lc) { return lc == lc ? (uint32_t)(-lc * 262144.0 + 0.5) : LC_NAN; }
// e^(Lc_t - Lc_j), t at or behind j
__device__ __forceinline__ float decay_of(uint32_t t, uint32_t j) {
    return __builtin_amdgcn_exp2f((float)(t - j) * (-LC_UNIT * 1.44269504088896341f));
}
// NaN for the sum up to a step behind a NaN one (A_log may be NaN)
__device__ __forceinline__ float nan_of(uint32_t lc) { return lc == LC_NAN ? NAN : 0.0f; }

// dt, the sums of A dt of every chunk and the walks' weights (from the sums in 64
// bits), zeros and the last sum behind the end: a wave a (chunk, head), two
// tokens a lane; the block's waves take neighbouring heads, whose dt lie
// together.
constexpr int ST_W = 4;
__global__ __launch_bounds__(ST_W * WAVE) void ssd_bwd_steps_kernel(SsdBwdArgs a) {
    const uint32_t c = blockIdx.x, h = blockIdx.y * ST_W + threadIdx.x / WAVE, b = blockIdx.z, lane = threadIdx.x % WAVE;
    if (h >= a.H) return;
    const double A = -exp((double)to_f(((const bf16*)a.A_log)[h]));
    const float bias = to_f(((const bf16*)a.dt_bias)[h]);
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
    f32x2 dt{0.0f, 0.0f}, slope{0.0f, 0.0f}, back, fwd;
    double s[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t t = c * FQ + 2 * lane + k;
        if (t < a.L) {
            const float v = to_f(((const bf16*)a.dt)[((size_t)b * a.L + t) * a.H + h]) + bias;
            const float sp = v > 20.0f ? v : log1pf(expf(v));
            dt[k] = fminf(fmaxf(sp, a.dt_min), a.dt_max);
            slope[k] = slope_of(a, v, sp);
        }
        s[k] = bounded(A * (double)dt[k]);
    }
    double before = s[0] + s[1];
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const double o = __shfl_up(before, d);
        if ((int)lane >= d) before += o;
    }
    const double last = __shfl(before, WAVE - 1);
    before = __shfl_up(before, 1);
    if (lane == 0) before = 0.0;
    s[0] += before;
    s[1] += s[0];
    uint2v lc;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        lc[k] = to_units(s[k]);
        back[k] = expf((float)s[k]);
        fwd[k] = dt[k] * expf((float)(last - s[k]));
    }
    const size_t at = (((size_t)b * a.H + h) * a.nchunk + c) * FQ + 2 * lane;
    *reinterpret_cast<uint2v*>(a.lc + at) = lc;
    *reinterpret_cast<f32x2*>(a.dtv + at) = dt;
    *reinterpret_cast<f32x2*>(a.slope + at) = slope;
    *reinterpret_cast<f32x2*>(a.w_back + at) = back;
    *reinterpret_cast<f32x2*>(a.w_fwd + at) = fwd;
}

// where tile (row tile, column tile) of a kept state's piece starts
__device__ __forceinline__ constexpr uint32_t state_at(uint32_t pt, uint32_t nt, uint32_t piece) {
    return ((pt * (FN / 16) + nt) * 2 + piece) * 256;
}

// The walk: block (head, slice, part of the state's columns), sequence,
// direction; wave w keeps the state's rows 16 w .. + 15, all NC columns of the
// part, in fp32.  A chunk's state goes out as two pieces, in tiles of 16 rows by
// 16 columns ([row tile][column tile][piece][n][row]): what a wave stores at
// once is contiguous (32 bytes of each of four waves to a line: 424 us where this
// takes 333, 4 x 4096 tokens), and a lane of the chunks' kernel finds its operand
// in 16 bytes.  A walk of 32 steps is latency at one sequence (111 us at 4096
// tokens, 320 blocks on 256 CUs: the waves issue 41 % of their cycles and wait for
// memory or LDS 24 %), and bandwidth and issue at four (296 us: 1.25 GB, 4.2
// TB/s; 310 us with the parts of a slice on two XCDs, which read its rows twice).  NC 32, 64, 128: 93, 86, 97 us at one sequence with the inputs in cache,
// 409, 300, 300 at four.
constexpr int W_NT = 256, NC = 64;
constexpr uint32_t XCDS = 8;
__global__ __launch_bounds__(W_NT, 3) void ssd_bwd_walk_bf16_kernel(SsdBwdArgs a) {
    constexpr int PARTS = FN / NC, NTL = NC / 16, BP = NC + 16;
    constexpr int XV = FQ * FP / 8 / W_NT, BV = FQ * NC / 8 / W_NT;     // 16-byte pieces a thread stages
    __shared__ __attribute__((aligned(16))) bf16 Xs[FQ * FXP], Bs[FQ * BP];
    __shared__ __attribute__((aligned(16))) float W[FQ];
    // The parts of a head's slice read the same rows: they are XCDS blocks apart,
    // which one XCD gets, and its L2 serves the second.
    const uint32_t all = a.H * a.nslice, first = blockIdx.x / (XCDS * PARTS) * XCDS, some = min(XCDS, all - first);
    const uint32_t at8 = blockIdx.x - first * PARTS, n0 = at8 / some * NC, hs = first + at8 % some;
    const uint32_t h = hs / a.nslice, sl = hs % a.nslice, b = blockIdx.y;
    const bool back = blockIdx.z != 0;
    const uint32_t P = a.P, L = a.L, g = h / (a.H / a.G), tid = threadIdx.x;
    const int lane = tid % WAVE, li = lane % 16, lq = lane / 16, tk = li / 4, tc = li % 4;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const float* init = back ? a.d_state : a.state;
    bf16* slots = (bf16*)(back ? a.gst : a.hst) + (((size_t)b * a.H + h) * a.nslice + sl) * a.nchunk * (2 * FN * FP);
    const bf16* rows = (const bf16*)(back ? a.dY : a.X) + (size_t)b * L * a.H * P + (size_t)h * P + sl * FP;
    const bf16* cols = (const bf16*)(back ? a.C : a.B) + (size_t)b * L * a.G * FN + (size_t)g * FN + n0;
    const float* weights = (back ? a.w_back : a.w_fwd) + ((size_t)b * a.H + h) * a.nchunk * FQ;
    const float* decays = a.w_back + ((size_t)b * a.H + h) * a.nchunk * FQ + FQ - 1;
    const size_t plain = (((size_t)b * a.H + h) * P + sl * FP + 16 * w + 4 * lq) * FN + n0 + li;

    floatx4 s[NTL];
#pragma unroll
    for (int i = 0; i < NTL; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = init ? init[plain + r * FN + 16 * i] : 0.0f;

    u32x4 rx[XV], rb[BV];
    float rw = 0.0f, rq = 0.0f;
    // the chunk's rows (behind the sequence's end, and for live = false: zeros,
    // as out of the resource's range)
    const uint32_t xat = tid / (FP / 8) * (a.H * P * 2) + tid % (FP / 8) * 16;
    const uint32_t bat = tid / (NC / 8) * (a.G * FN * 2) + tid % (NC / 8) * 16;
    auto fetch = [&](uint32_t c, bool live) {
        const uint32_t t0 = c * FQ, tl = min((uint32_t)FQ, L - t0);
        const auto xr = rsrc(rows + (size_t)t0 * a.H * P, live ? ((tl - 1) * a.H * P + FP) * 2 : 0);
        const auto br = rsrc(cols + (size_t)t0 * a.G * FN, live ? ((tl - 1) * a.G * FN + NC) * 2 : 0);
        const auto wr = rsrc(weights + t0, live ? FQ * 4 : 0), qr = rsrc(decays + t0, live ? 4 : 0);
#pragma unroll
        for (int i = 0; i < XV; ++i)
            rx[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, xat, i * (W_NT / (FP / 8)) * a.H * P * 2, 0);
#pragma unroll
        for (int i = 0; i < BV; ++i)
            rb[i] = __builtin_amdgcn_raw_buffer_load_b128(br, bat, i * (W_NT / (NC / 8)) * a.G * FN * 2, 0);
        rw = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(wr, tid % FQ * 4, 0, 0));
        rq = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(qr, 0, 0, 0));
    };
    // the state of chunk c (live = false: nowhere).  Issued behind the loads of
    // the next chunk, which are waited for without it
    auto put = [&](uint32_t c, bool live) {
        const auto r = rsrc(slots + (size_t)c * (2 * FN * FP), live ? 2 * FN * FP * 2 : 0);
        const uint32_t at = (state_at(w, n0 / 16, 0) + 16 * li + 4 * lq) * 2;
#pragma unroll
        for (int i = 0; i < NTL; ++i) {
            floatx4 v = s[i];
            const s4v hi = take4(v), lo = take4(v);
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, hi), r, at, state_at(0, i, 0) * 2, 0);
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, lo), r, at, state_at(0, i, 1) * 2, 0);
        }
    };
    if (a.nchunk) {
        fetch(back ? a.nchunk - 1 : 0, true);
        put(back ? a.nchunk - 1 : 0, true);
    }
    for (uint32_t k = 0; k < a.nchunk; ++k) {
        const uint32_t c = back ? a.nchunk - 1 - k : k;
        lds_barrier();
#pragma unroll
        for (int i = 0; i < XV; ++i) {
            const uint32_t j = tid + i * W_NT;
            *reinterpret_cast<u32x4*>(Xs + j / (FP / 8) * FXP + j % (FP / 8) * 8) = rx[i];
        }
#pragma unroll
        for (int i = 0; i < BV; ++i) {
            const uint32_t j = tid + i * W_NT;
            *reinterpret_cast<u32x4*>(Bs + j / (NC / 8) * BP + j % (NC / 8) * 8) = rb[i];
        }
        W[tid % FQ] = rw;      // (both halves of the block the same)
        const float dq = rq;
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NTL; ++i) s[i] *= dq;
        fetch(back ? max(c, 1u) - 1 : min(c + 1, a.nchunk - 1), k + 1 < a.nchunk);
        // The rows, weighted, in pieces: three backwards, as the gradient of the
        // first state is given in fp32; two forwards, where the states are only
        // kept as two.  A piece's products run while the next rows are split.
        auto split = [&](int ks, s8v (&f)[3]) {
            // k = token in the order 4 q .. + 3, 16 + 4 q .. + 3 of each 32:
            // the transposing loads meet no bank twice
            const bf16* xp = Xs + (32 * ks + 4 * lq + tk) * FXP + 16 * w + 4 * tc;
            const s4v x0 = ld_tr(xp), x1 = ld_tr(xp + 16 * FXP);
            floatx4 v0 = *reinterpret_cast<const floatx4*>(W + 32 * ks + 4 * lq);
            floatx4 v1 = *reinterpret_cast<const floatx4*>(W + 32 * ks + 16 + 4 * lq);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v0[e] *= val(x0[e]);
                v1[e] *= val(x1[e]);
            }
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                const s4v lo = take4(v0);
                f[e] = cat8(lo, take4(v1));
            }
        };
        auto products = [&](auto pieces) {
            s8v f[2][3];
            split(0, f[0]);
#pragma unroll
            for (int ks = 0; ks < FQ / 32; ++ks) {
                if (ks + 1 < FQ / 32) split(ks + 1, f[(ks + 1) % 2]);
#pragma unroll
                for (int i = 0; i < NTL; ++i) {
                    const bf16* bp = Bs + (32 * ks + 4 * lq + tk) * BP + 16 * i + 4 * tc;
                    const s8v bt = cat8(ld_tr(bp), ld_tr(bp + 16 * BP));
#pragma unroll
                    for (int e = 0; e < decltype(pieces)::value; ++e) s[i] = mma(f[ks % 2][e], bt, s[i]);
                }
            }
        };
        if (back) products(std::integral_constant<int, 3>{});
        else products(std::integral_constant<int, 2>{});
        put(back ? max(c, 1u) - 1 : min(c + 1, a.nchunk - 1), k + 1 < a.nchunk);
    }
    if (back && a.d_state0)
#pragma unroll
        for (int i = 0; i < NTL; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) a.d_state0[plain + r * FN + 16 * i] = s[i][r];
}

// The chunks' gradients: block = chunk, sequence, group, share of the group's
// (head, slice) pairs, which it takes one after the other.  Wave w
//   - keeps dB and dC of state columns 16 w .. + 15, all tokens, in registers;
//   - forms column J of S and M (source tokens 16 J .. + 15, all sinks), J such
//     that the two waves of a SIMD share nine of the 36 lower tiles, and from
//     it dx of those tokens; M goes from the registers that S came out in
//     into the next product.
// C B^T and the heads' sum of S (lower tiles, as their product leaves them) live
// in LDS.  The next pair's rows and states are on their way into registers
// while this one is worked on.
// No one thing bounds it: 450 us at 4 x 4096 tokens of 80 heads; 394 with all
// loads from the caches, 392 without S and M, 420 without dx' from G1, 441 without
// dC of what was before the chunk, and 194 with none of these and no dB: staging,
// barriers and dx in a row.  A wave issues 1256 VALU, 141 MFMA and 217 LDS
// instructions a pair (VALU 45 % of the SIMDs' cycles, MFMA 20 %).  Two tiles of S
// at a time need more than the 256 registers that two waves a SIMD leave (120 ->
// 213 us at 4096 tokens, with spills); the next pair's rows fetched before S, and
// B and h0 at the pair's start instead, came out even (457 and 464).
constexpr int F_TILES = 36;
__device__ __forceinline__ constexpr int tile_of(int T, int J) { return T * (T + 1) / 2 + J; }

// Sums over the 16 lanes of a row of four values each; lane i ends with that
// of value i % 4.
__device__ __forceinline__ float row_sums4(const floatx4& v) {
    const uint32_t l = threadIdx.x;
    const bool b0 = l & 1, b1 = l & 2;
    const float a = (b0 ? v[1] : v[0]) + dpp_f32<0xB1>(b0 ? v[0] : v[1]);      // values 0, 1
    const float c = (b0 ? v[3] : v[2]) + dpp_f32<0xB1>(b0 ? v[2] : v[3]);      // values 2, 3
    float s = (b1 ? c : a) + dpp_f32<0x4E>(b1 ? a : c);
    s += dpp_f32<0x124>(s);                                                    // row_ror:4
    return s + dpp_f32<0x128>(s);                                              // row_ror:8
}

__global__ __launch_bounds__(F_NT) void ssd_bwd_chunk_bf16_kernel(SsdBwdArgs a) {
    __shared__ __attribute__((aligned(16))) bf16 stage[4 * FQ * FXP];
    __shared__ __attribute__((aligned(16))) floatx4 SS[F_TILES * WAVE], CB[F_TILES * WAVE];
    __shared__ __attribute__((aligned(16))) float DT[FQ], EL[FQ], ER[FQ], WB[FQ], AF[FQ];
    __shared__ __attribute__((aligned(16))) uint32_t LC[FQ];
    __shared__ float SL[FQ], VO[8][FQ], RS[8][FQ], UO[FQ], CS[FQ], red[8][2], TL[6][FQ], TE[2];
    bf16 *Xs = stage, *Ys = stage + FQ * FXP, *Gh = stage + 2 * FQ * FXP, *Gl = stage + 3 * FQ * FXP;
    const uint32_t P = a.P, L = a.L, hpg = a.H / a.G;
    uint32_t tid = threadIdx.x;
    const uint32_t c = blockIdx.x % a.nchunk, sp = blockIdx.x / a.nchunk % a.nsplit;
    const uint32_t g = blockIdx.x / a.nchunk / a.nsplit, b = blockIdx.y;
    const uint32_t t0 = c * FQ, tl = min((uint32_t)FQ, L - t0);
    int lane = tid % WAVE, li = lane % 16, lq = lane / 16, tk = li / 4, tc = li % 4;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int J = w < 4 ? w : 11 - w;
    const size_t hp = (size_t)a.H * P, gn = (size_t)a.G * FN;
    const bf16* Bg = (const bf16*)a.B + ((size_t)b * L + t0) * gn + (size_t)g * FN;
    const bf16* Cg = (const bf16*)a.C + ((size_t)b * L + t0) * gn + (size_t)g * FN;

    const uint32_t pairs = hpg * a.nslice, per = (pairs + a.nsplit - 1) / a.nsplit;
    const uint32_t v_first = sp * per, v_end = min(pairs, v_first + per);
    u32x4 rx[2], ry[2], rg[4], rh[4];
    float rd = 0.0f, rs = 0.0f;
    uint32_t rl = 0, rt = 0, rr = 0, ra = 0, rD = 0;
    auto fetch = [&](uint32_t v, bool live) {
        const uint32_t h = g * hpg + v / a.nslice, sl = v % a.nslice;
        const size_t row0 = ((size_t)b * L + t0) * hp + (size_t)h * P + sl * FP;
        // rows behind the sequence's end are out of the resource's range: zeros
        const uint32_t range = live ? (uint32_t)(((tl - 1) * hp + FP) * sizeof(bf16)) : 0u, whole = live ? 2 * FN * FP * 2 : 0;
        const auto xr = rsrc((const bf16*)a.X + row0, range), yr = rsrc((const bf16*)a.dY + row0, range);
        const uint32_t step = (uint32_t)hp * (F_NT / (FP / 8) * sizeof(bf16));
        const uint32_t at = (tid / (FP / 8)) * (uint32_t)(hp * sizeof(bf16)) + tid % (FP / 8) * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            rx[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, at, i * step, 0);
            ry[i] = __builtin_amdgcn_raw_buffer_load_b128(yr, at, i * step, 0);
        }
        const size_t slot = ((((size_t)b * a.H + h) * a.nslice + sl) * a.nchunk + c) * (2 * FN * FP);
        const auto gr = rsrc((const bf16*)a.gst + slot, whole), hr = rsrc((const bf16*)a.hst + slot, whole);
        const uint32_t ha = (state_at(lq / 2, w, 0) + 16 * li + 8 * (lq % 2)) * 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            rg[i] = __builtin_amdgcn_raw_buffer_load_b128(gr, 16 * tid, i * F_NT * 16, 0);
            rh[i] = __builtin_amdgcn_raw_buffer_load_b128(hr, ha, state_at(2 * (i % 2), 0, i / 2) * 2, 0);
        }
        const size_t sp0 = (((size_t)b * a.H + h) * a.nchunk + c) * FQ;
        const uint32_t some = live ? FQ * 4 : 0, tt = tid % FQ;
        const auto lr = rsrc(a.lc + sp0, some), dr = rsrc(a.dtv + sp0, some), sr = rsrc(a.slope + sp0, some);
        auto one = [](auto r, uint32_t at) -> uint32_t { return __builtin_amdgcn_raw_buffer_load_b32(r, 4 * at, 0, 0); };
        rl = one(lr, tt);
        rt = one(lr, FQ - 1);
        rr = one(lr, tt >= 16 ? tt / 16 * 16 - 1 : 0);      // (token blocks past the first)
        rd = __uint_as_float(one(dr, tt));
        rs = __uint_as_float(one(sr, tt));
        ra = __builtin_amdgcn_raw_buffer_load_b16(rsrc((const bf16*)a.A_log + h, 2), 0, 0, 0);
        rD = __builtin_amdgcn_raw_buffer_load_b16(rsrc((const bf16*)a.D + h, a.D ? 2 : 0), 0, 0, 0);
    };

    auto touch = [&](uint32_t v, uint32_t (&out)[2]) {
        const uint32_t h = g * hpg + v / a.nslice, sl = v % a.nslice, r = min(tid % FQ, tl - 1);
        const size_t row = ((size_t)b * L + t0 + r) * hp + (size_t)h * P + sl * FP;
        const size_t slot = ((((size_t)b * a.H + h) * a.nslice + sl) * a.nchunk + c) * (2 * FN * FP);
        const bf16* first = tid < 2 * FQ ? (const bf16*)(tid < FQ ? a.X : a.dY) + row : (const bf16*)a.gst + slot + 64 * (tid - 2 * FQ);
        out[0] = *reinterpret_cast<const uint32_t*>(first);
        out[1] = *reinterpret_cast<const uint32_t*>((const bf16*)a.hst + slot + 64 * (tid % 256));
    };
    if (v_first < v_end) fetch(v_first, true);

    // B and C once through LDS: C B^T (lower tiles), B of the wave's sources, C
    // of its columns
    bf16 *Bs = stage, *Cs = stage + FQ * FBP;
    static_assert(2 * FBP <= 4 * FXP, "B and C fit where the pairs' tiles are");
    auto stage_bc = [&]() {
        const auto br = rsrc(Bg, ((tl - 1) * a.G * FN + FN) * 2), cr = rsrc(Cg, ((tl - 1) * a.G * FN + FN) * 2);
        u32x4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t j = tid + i * F_NT, at = j / (FN / 8) * (a.G * FN * 2) + j % (FN / 8) * 16;
            x[i] = __builtin_amdgcn_raw_buffer_load_b128(br, at, 0, 0);
            y[i] = __builtin_amdgcn_raw_buffer_load_b128(cr, at, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t j = tid + i * F_NT, at = j / (FN / 8) * FBP + j % (FN / 8) * 8;
            *reinterpret_cast<u32x4*>(Bs + at) = x[i];
            *reinterpret_cast<u32x4*>(Cs + at) = y[i];
        }
    };
    stage_bc();
    lds_barrier();
    for (int i = w; i < F_TILES; i += 8) {
        int T = 0;
        while (tile_of(T + 1, 0) <= i) ++T;
        const bf16 *cr = Cs + (16 * T + li) * FBP + 8 * lq, *br = Bs + (16 * (i - tile_of(T, 0)) + li) * FBP + 8 * lq;
        floatx4 acc{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < FN / 32; ++ks)
            acc = mma(*reinterpret_cast<const s8v*>(cr + 32 * ks), *reinterpret_cast<const s8v*>(br + 32 * ks), acc);
        CB[i * WAVE + lane] = acc;
        SS[i * WAVE + lane] = floatx4{0, 0, 0, 0};
    }
    RS[w][lane] = RS[w][lane + 64] = 0.0f;      // sinks before the wave's sources stay 0
    // k = n in the order 4 q .. + 3, 16 + 4 q .. + 3 of each 32, in which the
    // transposing loads of the other operand meet no bank twice
    s8v bf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        const bf16* br = Bs + (16 * J + li) * FBP + 32 * ks + 4 * lq;
        bf[ks] = cat8(*reinterpret_cast<const s4v*>(br), *reinterpret_cast<const s4v*>(br + 16));
    }
    s4v cp[8];                                   // C[t = 16 T + li][n = 16 w + 4 lq + r]
#pragma unroll
    for (int T = 0; T < 8; ++T) cp[T] = *reinterpret_cast<const s4v*>(Cs + (16 * T + li) * FBP + 16 * w + 4 * lq);

    floatx4 dc[8], db[8];                        // [n = 16 w + 4 lq + r][t = 16 T + li]
#pragma unroll
    for (int T = 0; T < 8; ++T) dc[T] = db[T] = floatx4{0, 0, 0, 0};

    // a_t: pairs of a source before t and a sink from t on; lane l has tokens
    // 2 l and 2 l + 1.  The wave with the fewest tiles gathers a pair's sums and
    // finishes them while the others work on the next.
    constexpr int TAIL = 4;
    float tA = 0.0f;
    auto gather = [&]() {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int t = 2 * lane + k;
            float suf = 0.0f, in = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) suf += VO[i][t];
#pragma unroll
            for (int i = 0; i < 8; ++i) in += RS[i][t];
            const float dt = DT[t], u = UO[t];
            TL[0][t] = dt * u;
            TL[1][t] = suf;
            TL[2][t] = in;
            TL[3][t] = u + CS[t];
            TL[4][t] = dt;
            TL[5][t] = SL[t];
        }
        float tedge = 0.0f, tdd = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            tedge += red[i][0];
            tdd += red[i][1];
        }
        if (lane < 2) TE[lane] = lane ? tdd : tedge * EL[FQ - 1];
    };
    auto finish = [&](uint32_t v) {
        const uint32_t h = g * hpg + v / a.nslice, sl = v % a.nslice;
        float pre[2], suf[2], in[2], dir[2], tdt[2], tsl[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int t = 2 * lane + k;
            pre[k] = TL[0][t];
            suf[k] = TL[1][t];
            in[k] = TL[2][t];
            dir[k] = TL[3][t];
            tdt[k] = TL[4][t];
            tsl[k] = TL[5][t];
        }
        const float tedge = TE[0], tdd = TE[1];
        // sums before and behind this lane's tokens (not as differences of
        // longer ones: a step that forgets leaves far less than there was)
        float before = __shfl_up(wave_prefix_sum(pre[0] + pre[1]), 1);
        if (lane == 0) before = 0.0f;
        float behind = __shfl(wave_prefix_sum(__shfl(suf[0] + suf[1], 63 - lane)), 62 - lane);
        if (lane == 63) behind = 0.0f;
        before += tedge;
        behind += suf[1];
        const float da0 = before + ((behind + suf[0]) + in[0]), da1 = (before + pre[0]) + (behind + in[1]);
        const float q0 = fmaf(tA, da0, dir[0]) * tsl[0], q1 = fmaf(tA, da1, dir[1]) * tsl[1];
        float* q = a.q + (((size_t)sl * a.batch + b) * a.H + h) * L + t0;
        if (2 * lane < (int)tl) q[2 * lane] = q0;
        if (2 * lane + 1 < (int)tl) q[2 * lane + 1] = q1;
        const float dA = wave_sum(tdt[0] * da0 + tdt[1] * da1), dq = wave_sum(q0 + q1);
        if (lane == 0) {
            float* o = a.part + ((((size_t)b * a.H + h) * a.nslice + sl) * a.nchunk + c) * 3;
            o[0] = dq;
            o[1] = tA * dA;
            o[2] = tdd;
        }
    };

    for (uint32_t v = v_first; v < v_end; ++v) {
        const uint32_t h = g * hpg + v / a.nslice, sl = v % a.nslice;
        // places and C's values are formed again for each pair: kept over the
        // loop they would push what has to be kept out of the registers
        asm volatile("" : "+v"(tid), "+v"(lane), "+v"(li), "+v"(lq), "+v"(tk), "+v"(tc));
#pragma unroll
        for (int T = 0; T < 8; ++T) asm volatile("" : "+v"(cp[T]));
        lds_barrier();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t j = tid + i * F_NT, at = j / (FP / 8) * FXP + j % (FP / 8) * 8;
            *reinterpret_cast<u32x4*>(Xs + at) = rx[i];
            *reinterpret_cast<u32x4*>(Ys + at) = ry[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // 16 bytes j of the state: 32 a tile's piece
            const uint32_t j = tid + i * F_NT, pc = j / 32 % 2, nt = j / 64 % (FN / 16), pt = j / 64 / (FN / 16);
            *reinterpret_cast<u32x4*>((pc ? Gl : Gh) + (16 * nt + j % 32 / 2) * FXP + 16 * pt + 8 * (j % 2)) = rg[i];
        }
        const float D = val((short)rD), A_h = -__expf(val((short)ra));
        if (tid < FQ) {
            const float er = decay_of(rt, rl) + nan_of(rt);
            LC[tid] = rl;
            DT[tid] = rd;
            EL[tid] = decay_of(rl, 0) + nan_of(rl);
            ER[tid] = er;
            WB[tid] = rd * er;
            AF[tid] = decay_of(rl, rr);
            SL[tid] = rs;
        }
        lds_barrier();
        // one word of each line of the next pair's rows and states, long before
        // the registers that take them are free: they come from the L2 then
        uint32_t touched[2] = {0, 0};
        if (v + 1 < v_end) touch(v + 1, touched);
        if (w == TAIL && v > v_first) finish(v - 1);
        tA = A_h;

        // dB^T [n][source]: G1 and x (k = row); <G1, h0> as a trace
        s8v gf[4], hf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gf[i] = *reinterpret_cast<const s8v*>((i / 2 ? Gl : Gh) + (16 * w + li) * FXP + 32 * (i % 2) + 8 * lq);
            hf[i] = __builtin_bit_cast(s8v, rh[i]);
        }
        floatx4 tr{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            tr = mma(gf[ks], hf[ks], tr);
            tr = mma(gf[ks], hf[ks + 2], tr);
            tr = mma(gf[ks + 2], hf[ks], tr);
        }
#pragma unroll
        for (int T = 0; T < 8; ++T) {
            const bf16* xp = Xs + (16 * T + li) * FXP + 8 * lq;
            const s8v x0 = *reinterpret_cast<const s8v*>(xp), x1 = *reinterpret_cast<const s8v*>(xp + 32);
            floatx4 y{0, 0, 0, 0};
            y = mma(gf[0], x0, y);
            y = mma(gf[1], x1, y);
            y = mma(gf[2], x0, y);
            y = mma(gf[3], x1, y);
            const float wb = WB[16 * T + li];
#pragma unroll
            for (int r = 0; r < 4; ++r) db[T][r] = fmaf(wb, y[r], db[T][r]);
        }
        float gh = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) gh += 4 * lq + r == li ? tr[r] : 0.0f;

        // dx'^T [row][source] from G1 and B (k = n)
        const int j = 16 * J + li;
        floatx4 dx[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) dx[p] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int at = (32 * ks + 4 * lq + tk) * FXP + 16 * p + 4 * tc;
                dx[p] = mma(cat8(ld_tr(Gh + at), ld_tr(Gh + at + 16 * FXP)), bf[ks], dx[p]);
                dx[p] = mma(cat8(ld_tr(Gl + at), ld_tr(Gl + at + 16 * FXP)), bf[ks], dx[p]);
            }
        const float erj = ER[j], dtj = DT[j];
        const uint32_t lcj = LC[j];
        float uo = 0.0f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const s4v x = *reinterpret_cast<const s4v*>(Xs + j * FXP + 16 * p + 4 * lq);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                dx[p][r] *= erj;
                uo = fmaf(dx[p][r], val(x[r]), uo);
            }
        }
        uo = swap_add32(swap_add16(uo));

        // sinks T: dC^T [n][sink] of all sources before the chunk; S and M of column J
        const s8v xj0 = *reinterpret_cast<const s8v*>(Xs + j * FXP + 8 * lq);
        const s8v xj1 = *reinterpret_cast<const s8v*>(Xs + j * FXP + 32 + 8 * lq);
        float col = 0.0f, diag = 0.0f, below = 0.0f;
#pragma unroll
        for (int T2 = 6; T2 >= 0; T2 -= 2) {
            s4v mh[2], ml[2];
#pragma unroll
            for (int k = 1; k >= 0; --k) {
                const int T = T2 + k;
                const bf16* yp = Ys + (16 * T + li) * FXP + 8 * lq;
                const s8v y0 = *reinterpret_cast<const s8v*>(yp), y1 = *reinterpret_cast<const s8v*>(yp + 32);
                floatx4 x{0, 0, 0, 0};
                x = mma(hf[0], y0, x);
                x = mma(hf[1], y1, x);
                x = mma(hf[2], y0, x);
                x = mma(hf[3], y1, x);
                const float el = EL[16 * T + li];
                float vo = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    dc[T][r] = fmaf(el, x[r], dc[T][r]);
                    vo = fmaf(x[r], val(cp[T][r]), vo);
                }
                vo = el * swap_add32(swap_add16(vo));
                if (lq == 0) VO[w][16 * T + li] = vo;
                mh[k] = ml[k] = s4v{0, 0, 0, 0};
                if (T >= J) {
                    floatx4 sd{0, 0, 0, 0};
                    sd = mma(y0, xj0, sd);
                    sd = mma(y1, xj1, sd);
                    const int id = tile_of(T, 0) + J;
                    floatx4 e;
                    if (T > J) {
                        const float f = decay_of(LC[16 * T - 1], lcj);
                        e = *reinterpret_cast<const floatx4*>(AF + 16 * T + 4 * lq) * f;
                    } else {
                        const u32x4 lt = *reinterpret_cast<const u32x4*>(LC + 16 * T + 4 * lq);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            e[r] = 4 * lq + r >= li ? decay_of(lt[r], lcj) : 0.0f;
                            diag += 4 * lq + r == li ? sd[r] : 0.0f;
                        }
                    }
                    const floatx4 cb = CB[id * WAVE + lane];
                    floatx4 ss = SS[id * WAVE + lane], m, row;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float se = sd[r] * e[r], sdt = se * dtj;
                        m[r] = cb[r] * e[r];
                        ss[r] += sdt;
                        col = fmaf(se, cb[r], col);
                        row[r] = sdt * cb[r];
                    }
                    SS[id * WAVE + lane] = ss;
                    // sinks from t on, this wave's sources before t
                    if (T == J)
#pragma unroll
                        for (int r = 0; r < 4; ++r) row[r] = 4 * lq + r > li ? row[r] : 0.0f;
                    from_row(row, below);
                    if (T == J)
#pragma unroll
                        for (int r = 0; r < 4; ++r) row[r] = 4 * lq + r > li ? row[r] : 0.0f;
                    const float rsum = row_sums4(row);
                    if (li < 4) RS[w][16 * T + 4 * lq + li] = rsum;
                    mh[k] = take4(m);
                    ml[k] = take4(m);
                }
            }
            if (T2 + 1 >= J) {
                const s8v h8 = cat8(mh[0], mh[1]), l8 = cat8(ml[0], ml[1]);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const bf16* yp = Ys + (16 * T2 + 4 * lq + tk) * FXP + 16 * p + 4 * tc;
                    const s8v yt = cat8(ld_tr(yp), ld_tr(yp + 16 * FXP));
                    dx[p] = mma(yt, h8, dx[p]);
                    dx[p] = mma(yt, l8, dx[p]);
                }
            }
        }
        col = swap_add32(swap_add16(col));
        if (lq == 0) {
            UO[j] = uo;
            CS[j] = col;
        }
        gh = wave_sum(gh);
        diag = wave_sum(diag);
        if (lane == 0) {
            red[w][0] = gh;
            red[w][1] = diag;
        }
        bf16* out0 = (bf16*)a.dX + ((size_t)b * L + t0) * hp + (size_t)h * P + sl * FP;
        const uint32_t out = j * (uint32_t)hp + 4 * lq;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const s4v y = *reinterpret_cast<const s4v*>(Ys + j * FXP + 16 * p + 4 * lq);
            floatx4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(dtj, dx[p][r], D * val(y[r]));
            if (j < (int)tl) *reinterpret_cast<s4v*>(out0 + (out + 16 * p)) = take4(o);
        }
        // behind the stores: waiting for the next pair at the top waits for
        // nothing that was issued later
        asm volatile("" ::"v"(touched[0]), "v"(touched[1]));
        fetch(min(v + 1, v_end - 1), v + 1 < v_end);
        lds_barrier();
        if (w == TAIL) gather();
    }
    if (w == TAIL && v_first < v_end) finish(v_end - 1);

    // within the chunk: sum of S over the share's heads with B and C
    lds_barrier();
    stage_bc();
    lds_barrier();
    const float* Sf = reinterpret_cast<const float*>(SS);
#pragma unroll
    for (int T = 0; T < 8; ++T) {
        // dB of source tile T: sinks k = T ..; dC of sink tile T: sources k = .. T
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            const bf16* tp = (Cs + (16 * k + 4 * lq + tk) * FBP + 16 * w + 4 * tc);
            if (k + 1 >= T) {
                s4v hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    floatx4 x{0, 0, 0, 0};
                    if (k + e >= T) x = SS[(tile_of(k + e, 0) + T) * WAVE + lane];
                    hi[e] = take4(x);
                    lo[e] = take4(x);
                }
                const s8v ct = cat8(ld_tr(tp), ld_tr(tp + 16 * FBP));
                db[T] = mma(ct, cat8(hi[0], hi[1]), db[T]);
                db[T] = mma(ct, cat8(lo[0], lo[1]), db[T]);
            }
            if (k <= T) {
                const bf16* bp = (Bs + (16 * k + 4 * lq + tk) * FBP + 16 * w + 4 * tc);
                s4v hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    floatx4 x{0, 0, 0, 0};
                    if (k + e <= T)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            x[r] = Sf[((tile_of(T, 0) + k + e) * WAVE + 4 * lq + r + 16 * tk) * 4 + tc];
                    hi[e] = take4(x);
                    lo[e] = take4(x);
                }
                const s8v bt = cat8(ld_tr(bp), ld_tr(bp + 16 * FBP));
                dc[T] = mma(bt, cat8(hi[0], hi[1]), dc[T]);
                dc[T] = mma(bt, cat8(lo[0], lo[1]), dc[T]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const uint32_t t = 16 * T + li;
        if (t < tl) {
            const size_t at = (size_t)sp * a.share + (((size_t)b * L + t0 + t) * a.G + g) * FN + 16 * w + 4 * lq;
            *reinterpret_cast<floatx4*>(a.cpart + at) = dc[T];
            *reinterpret_cast<floatx4*>(a.bpart + at) = db[T];
        }
    }
}

// ---------------------------------------------------------------------------
// Sums over shares, slices and chunks
// ---------------------------------------------------------------------------
// One launch: blocks of four dB and dC elements a thread, then blocks of 64
// tokens by 16 heads of d_dt (which the chunks left a head at a time), then a
// block a head for the parameters' gradients, summed in 64 bits.
constexpr int R_NT = 256, R_T = 64, R_H = 16;

template <typename T> __device__ __forceinline__ void store4(T* dst, size_t i, size_t n, const float (&v)[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (i + 4 <= n && (uintptr_t)dst % sizeof(T4) == 0) {
        *reinterpret_cast<T4*>(dst + i) = T4{from_f<T>(v[0]), from_f<T>(v[1]), from_f<T>(v[2]), from_f<T>(v[3])};
    } else {
        for (int e = 0; e < 4 && i + e < n; ++e) dst[i + e] = from_f<T>(v[e]);
    }
}

template <typename T> __global__ __launch_bounds__(R_NT) void ssd_bwd_finish_kernel(SsdBwdArgs a) {
    __shared__ union {
        float tile[R_T][R_H + 1];
        double red[3][R_NT];
    } sh;
    const uint32_t tid = threadIdx.x;
    uint32_t blk = blockIdx.x;
    if (blk < a.row_blocks) {
        const size_t n = (size_t)a.batch * a.L * a.G * a.N, i = ((size_t)blk * R_NT + tid) * 4;
        if (i >= n) return;
        float x[4] = {}, y[4] = {};
#pragma unroll 8
        for (uint32_t s = 0; s < a.nsplit; ++s) {
            const floatx4 u = *reinterpret_cast<const floatx4*>(a.bpart + s * a.share + i);
            const floatx4 v = *reinterpret_cast<const floatx4*>(a.cpart + s * a.share + i);
            for (int e = 0; e < 4; ++e) {
                x[e] += u[e];
                y[e] += v[e];
            }
        }
        store4((T*)a.dB, i, n, x);
        store4((T*)a.dC, i, n, y);
        return;
    }
    blk -= a.row_blocks;
    if (blk < a.dt_blocks) {
        const uint32_t nh = (a.H + R_H - 1) / R_H, nt = (a.L + R_T - 1) / R_T;
        const uint32_t h0 = blk % nh * R_H, t0 = blk / nh % nt * R_T, b = blk / nh / nt;
        for (uint32_t i = tid; i < R_T * R_H; i += R_NT) {
            const uint32_t h = i / R_T, t = i % R_T;
            if (h0 + h >= a.H || t0 + t >= a.L) continue;
            float v = 0.0f;
            for (uint32_t s = 0; s < a.nslice; ++s) v += a.q[(((size_t)s * a.batch + b) * a.H + h0 + h) * a.L + t0 + t];
            sh.tile[t][h] = v;
        }
        __syncthreads();
        for (uint32_t i = tid; i < R_T * R_H; i += R_NT) {
            const uint32_t t = i / R_H, h = i % R_H;
            if (h0 + h < a.H && t0 + t < a.L) ((T*)a.d_dt)[((size_t)b * a.L + t0 + t) * a.H + h0 + h] = from_f<T>(sh.tile[t][h]);
        }
        return;
    }
    const uint32_t h = blk - a.dt_blocks;
    double s[3] = {0, 0, 0};
    const size_t np = (size_t)a.nslice * a.nchunk;
    for (size_t i = tid; i < a.batch * np; i += R_NT) {
        const float* o = a.part + (((size_t)(i / np) * a.H + h) * np + i % np) * 3;
        for (int k = 0; k < 3; ++k) s[k] += (double)o[k];
    }
    for (int k = 0; k < 3; ++k) sh.red[k][tid] = s[k];
    __syncthreads();
    for (int d = R_NT / 2; d; d >>= 1) {
        if ((int)tid < d)
            for (int k = 0; k < 3; ++k) sh.red[k][tid] += sh.red[k][tid + d];
        __syncthreads();
    }
    if (tid == 0) {
        ((T*)a.d_dt_bias)[h] = from_f<T>((float)sh.red[0][0]);
        ((T*)a.dA_log)[h] = from_f<T>((float)sh.red[1][0]);
        if (a.dD) ((T*)a.dD)[h] = from_f<T>((float)sh.red[2][0]);
    }
}

template <typename F> hipError_t with_type(int act, F f) {
    if (act == LSSM_BF16) return f(bf16{});
    if (act == LSSM_F16) return f(f16{});
    return f(float{});
}

// The plan and the workspace: [h0 states][G1 states][dB parts][dC parts][q][head parts][5 x steps]
struct Plan {
    bool fast;
    uint32_t nchunk, nslice, nsplit;
    size_t states, share, q, part, steps;      // floats of one of each
    size_t floats() const { return 2 * states + 2 * nsplit * share + q + part + 5 * steps; }
};
Plan plan_of(uint32_t batch, const lssm_ssd_dims& d, bool fast) {
    Plan p;
    p.fast = fast;
    const uint32_t qn = fast ? FQ : GQ, rn = fast ? FP : GP;
    p.nchunk = (d.L + qn - 1) / qn;
    p.nslice = (d.P + rn - 1) / rn;
    // shares of a group's (head, slice) pairs: the fewest rounds of blocks
    // over the chip, a block's own work taken as two pairs more (as none: 16
    // heads of N = 64, 2 x 1777 tokens 125 -> 147 us; as six: all alike)
    const uint32_t pairs = d.H / d.n_groups * p.nslice;
    const size_t blocks = std::max<size_t>(1, (size_t)p.nchunk * batch * d.n_groups), cus = (fast ? 1 : 2) * (size_t)num_cus();
    size_t best = 0;
    p.nsplit = 1;
    for (uint32_t per = pairs; per >= 1; --per) {
        const uint32_t n = (pairs + per - 1) / per;
        const size_t cost = (blocks * n + cus - 1) / cus * (per + 2);
        if (per == pairs || cost < best) {
            best = cost;
            p.nsplit = n;
        }
    }
    p.states = (size_t)batch * d.H * p.nchunk * d.P * d.N;
    p.share = (size_t)batch * d.L * d.n_groups * d.N;
    p.q = (size_t)p.nslice * batch * d.H * d.L;
    p.part = (size_t)batch * d.H * p.nslice * p.nchunk * 3;
    p.steps = (size_t)batch * d.H * p.nchunk * (fast ? FQ : 1);
    // every array starts on a 16-byte address
    for (size_t* n : {&p.states, &p.share, &p.q, &p.part, &p.steps}) *n = (*n + 3) / 4 * 4;
    return p;
}
// (the threads of a launch's x count in 32 bits)
bool launches(uint32_t batch, const lssm_ssd_dims& d, const Plan& p) {
    const uint64_t rows = (p.share + 4 * R_NT - 1) / (4 * R_NT);
    const uint64_t dts = (uint64_t)batch * ((d.L + R_T - 1) / R_T) * ((d.H + R_H - 1) / R_H);
    return (uint64_t)p.nchunk * p.nsplit * d.n_groups * F_NT < (1ull << 32) && (rows + dts + d.H) * R_NT < (1ull << 32);
}
// (a chunk's rows within 32-bit byte offsets)
bool fast_dims(const lssm_ssd_dims& d, int act) {
    return act == LSSM_BF16 && d.N == FN && d.P % FP == 0 && (uint64_t)d.H * std::max(d.P, d.N) * FQ * 2 < (1u << 31);
}

template <typename T, int NT> void launch_generic(hipStream_t s, const SsdBwdArgs& a) {
    if (a.nchunk) ssd_bwd_own_kernel<T, NT><<<dim3(a.H * a.nslice * 2, a.nchunk, a.batch), G_NT, 0, s>>>(a);
    ssd_bwd_scan_kernel<<<dim3((a.P * a.N + G_NT - 1) / G_NT * 2, a.H, a.batch), G_NT, 0, s>>>(a);
    if (a.nchunk)
        ssd_bwd_chunk_kernel<T, NT, NT == 64 ? 4 : 8><<<dim3(a.nchunk * a.nsplit * a.G, a.batch), NT == 64 ? 256 : 512, 0, s>>>(a);
}

}  // namespace

bool ssd_bwd_launches(uint32_t batch, const lssm_ssd_dims& d, int act) {
    return launches(batch, d, plan_of(batch, d, false)) && (!fast_dims(d, act) || launches(batch, d, plan_of(batch, d, true)));
}

// (the larger of both plans: alignment of the arrays decides at the call)
size_t ssd_bwd_ws_bytes(uint32_t batch, const lssm_ssd_dims& d, int act) {
    size_t n = plan_of(batch, d, false).floats();
    if (fast_dims(d, act)) n = std::max(n, plan_of(batch, d, true).floats());
    return n * sizeof(float);
}

hipError_t launch_ssd_bwd(hipStream_t s, SsdBwdArgs a, const lssm_ssd_dims& d, int act, void* ws) {
    bool fast = fast_dims(d, act);
    for (const void* p : {a.X, a.B, a.C, a.dY, (const void*)a.dX}) fast = fast && (uintptr_t)p % 16 == 0;
    const Plan p = plan_of(a.batch, d, fast);
    a.nchunk = p.nchunk;
    a.nslice = p.nslice;
    a.nsplit = p.nsplit;
    a.hst = static_cast<float*>(ws);
    a.gst = a.hst + p.states;
    a.bpart = a.gst + p.states;
    a.cpart = a.bpart + p.nsplit * p.share;
    a.q = a.cpart + p.nsplit * p.share;
    a.part = a.q + p.q;
    a.lc = a.part + p.part;
    a.dtv = a.lc + p.steps;
    a.slope = a.dtv + p.steps;
    a.w_fwd = a.slope + p.steps;
    a.w_back = a.w_fwd + p.steps;
    a.share = p.share;
    a.row_blocks = (uint32_t)((p.share + 4 * R_NT - 1) / (4 * R_NT));
    a.dt_blocks = a.batch * ((a.L + R_T - 1) / R_T) * ((a.H + R_H - 1) / R_H);
    return with_type(act, [&](auto z) {
        using T = decltype(z);
        if (a.batch) {
            if (fast) {
                if (a.nchunk) ssd_bwd_steps_kernel<<<dim3(a.nchunk, (a.H + ST_W - 1) / ST_W, a.batch), ST_W * WAVE, 0, s>>>(a);
                ssd_bwd_walk_bf16_kernel<<<dim3(a.H * a.nslice * (FN / NC), a.batch, 2), W_NT, 0, s>>>(a);
                if (a.nchunk)
                    ssd_bwd_chunk_bf16_kernel<<<dim3(a.nchunk * a.nsplit * a.G, a.batch), F_NT, 0, s>>>(a);
            } else if (a.N <= 64) launch_generic<T, 64>(s, a);
            else if (a.N <= 128) launch_generic<T, 128>(s, a);
            else launch_generic<T, 256>(s, a);
        }
        ssd_bwd_finish_kernel<T><<<a.row_blocks + a.dt_blocks + a.H, R_NT, 0, s>>>(a);
        return hipGetLastError();
    });
}

}  // namespace lssm
