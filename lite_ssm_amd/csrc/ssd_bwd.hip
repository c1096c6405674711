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
// which adds terms of one chunk only: no sum over the whole sequence cancels.
//
// Three steps: a walk over the chunks keeps the states h0 (forwards) and G1
// (backwards) of every chunk; the chunks' gradients, in parallel; sums over
// heads, slices and chunks.  Every order of summation is fixed.
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
// The sums of A dt are held in 64 bits: differences of sums that grow along a
// chunk are what every decay is the exponential of.
// ---------------------------------------------------------------------------
constexpr int GQ = 32;      // tokens a chunk
constexpr int GP = 32;      // state rows a slice
constexpr int GXP = 36;     // LDS pitch of a [token][row] tile (= 4 modulo 64 banks x 9)
constexpr int G_NT = 256;

struct Steps { double lc, tot; float dt; };

// dt and the sums of A dt of a chunk of GQ tokens, lane t of a wave (lanes
// past GQ repeat the last token's).
template <typename T> __device__ __forceinline__ Steps chunk_steps(const SsdBwdArgs& a, uint32_t b, uint32_t h, uint32_t t0,
                                                                   uint32_t tl) {
    const uint32_t t = threadIdx.x % WAVE;
    const double A = -exp((double)to_f(((const T*)a.A_log)[h]));
    double dt = 0.0;
    if (t < tl) {
        const double v = (double)to_f(((const T*)a.dt)[((size_t)b * a.L + t0 + t) * a.H + h]) +
                         (double)to_f(((const T*)a.dt_bias)[h]);
        dt = v > 40.0 ? v : log1p(exp(v));
        dt = fmin(fmax(dt, (double)a.dt_min), (double)a.dt_max);
    }
    double s = A * dt;
#pragma unroll
    for (int d = 1; d < GQ; d <<= 1) {
        const double o = __shfl_up(s, d);
        if ((int)t >= d) s += o;
    }
    return {s, __shfl(s, GQ - 1), (float)dt};
}

// rows t0 .. t0 + tl of a [rows][stride] array, columns c0 .. c0 + n, into
// LDS [GQ][pitch], zeros behind the ends (W columns in all)
template <typename T, int W> __device__ __forceinline__ void load_tile(float* dst, int pitch, const T* src, size_t stride,
                                                                       uint32_t rows, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < GQ * W; i += G_NT) {
        const uint32_t r = i / W, c = i % W;
        dst[r * pitch + c] = (r < rows && c < n) ? to_f(src[r * stride + c]) : 0.0f;
    }
}

// The walk: block (head, slice), sequence, direction.  Direction 0 keeps h0 of
// every chunk, 1 its G1; both add to the state weighted outer products of the
// chunk's rows (x with B, dy with C).
template <typename T, int NT> __global__ __launch_bounds__(G_NT) void ssd_bwd_walk_kernel(SsdBwdArgs a) {
    constexpr int NP = NT + 4, TN = NT / 64;
    __shared__ float Rs[GQ * GXP], Cs[GQ * NP], W[GQ], Dq;
    const uint32_t h = blockIdx.x / a.nslice, p0 = blockIdx.x % a.nslice * GP, b = blockIdx.y;
    const bool back = blockIdx.z != 0;
    const uint32_t P = a.P, N = a.N, L = a.L, pn = min((uint32_t)GP, P - p0);
    const uint32_t g = h / (a.H / a.G);
    const int tid = threadIdx.x, lane = tid % WAVE, li = lane % 16, lq = lane / 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const float* init = back ? a.d_state : a.state;
    float* slots = (back ? a.gst : a.hst) + ((size_t)b * a.H + h) * a.nchunk * P * N;
    floatx4 s[2][TN];
    auto each = [&](auto f) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t p = 16 * pt + 4 * lq + r, n = 16 * (w + 4 * i) + li;
                    s[pt][i][r] = (p < pn && n < N) ? f(s[pt][i][r], (size_t)(p0 + p) * N + n) : 0.0f;
                }
    };
    each([&](float, size_t at) { return init ? init[((size_t)b * a.H + h) * P * N + at] : 0.0f; });
    for (uint32_t k = 0; k < a.nchunk; ++k) {
        const uint32_t c = back ? a.nchunk - 1 - k : k, t0 = c * GQ, tl = min((uint32_t)GQ, L - t0);
        each([&](float v, size_t at) { return slots[(size_t)c * P * N + at] = v; });
        __syncthreads();
        load_tile<T, GP>(Rs, GXP, (const T*)(back ? a.dY : a.X) + ((size_t)b * L + t0) * a.H * P + (size_t)h * P + p0,
                         (size_t)a.H * P, tl, pn);
        load_tile<T, NT>(Cs, NP, (const T*)(back ? a.C : a.B) + ((size_t)b * L + t0) * a.G * N + (size_t)g * N,
                         (size_t)a.G * N, tl, N);
        if (w == 0) {
            const Steps st = chunk_steps<T>(a, b, h, t0, tl);
            if (lane < GQ) W[lane] = back ? (float)exp(st.lc) : st.dt * (float)exp(st.tot - st.lc);
            if (lane == 0) Dq = (float)exp(st.tot);
        }
        __syncthreads();
        const float dq = Dq;
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                s[pt][i] *= dq;
#pragma unroll
                for (int kk = 0; kk < GQ / 4; ++kk) {
                    const int t = 4 * kk + lq;
                    s[pt][i] = mma4(Rs[t * GXP + 16 * pt + li] * W[t], Cs[t * NP + 16 * (w + 4 * i) + li], s[pt][i]);
                }
            }
    }
    if (back && a.d_state0) each([&](float v, size_t at) { return a.d_state0[((size_t)b * a.H + h) * P * N + at] = v; });
}

// The chunks' gradients: block = chunk, sequence, group, share of the group's
// (head, slice) pairs.  dB and dC of the share stay in registers.
template <typename T, int NT> __global__ __launch_bounds__(G_NT) void ssd_bwd_chunk_kernel(SsdBwdArgs a) {
    constexpr int NP = NT + 4, TN = NT / 64;
    __shared__ float Bs[GQ * NP], Cs[GQ * NP], Hs[GP * NP], Gs[GP * NP];
    __shared__ float Xs[GQ * GXP], Ys[GQ * GXP], Ms[GQ * GXP];
    __shared__ double Lc[GQ];
    __shared__ float DT[GQ], EL[GQ], ER[GQ], RS[2][GQ], CS[2][GQ], VO[4][GQ], UO[2][GQ], red[4][2];
    const uint32_t P = a.P, N = a.N, L = a.L, hpg = a.H / a.G;
    const uint32_t c = blockIdx.x % a.nchunk, sp = blockIdx.x / a.nchunk % a.nsplit;
    const uint32_t g = blockIdx.x / a.nchunk / a.nsplit, b = blockIdx.y;
    const uint32_t t0 = c * GQ, tl = min((uint32_t)GQ, L - t0);
    const int tid = threadIdx.x, lane = tid % WAVE, li = lane % 16, lq = lane / 16;
    const int w = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int T0 = w / 2, J0 = w % 2;      // this wave's tile of S, M (tokens) and of dx (tokens T0, rows J0)

    load_tile<T, NT>(Bs, NP, (const T*)a.B + ((size_t)b * L + t0) * a.G * N + (size_t)g * N, (size_t)a.G * N, tl, N);
    load_tile<T, NT>(Cs, NP, (const T*)a.C + ((size_t)b * L + t0) * a.G * N + (size_t)g * N, (size_t)a.G * N, tl, N);
    __syncthreads();
    floatx4 cb{0, 0, 0, 0};
    for (int k = 0; k < NT / 4; ++k)
        cb = mma4(Cs[(16 * T0 + li) * NP + 4 * k + lq], Bs[(16 * J0 + li) * NP + 4 * k + lq], cb);

    floatx4 dc[2][TN], db[2][TN], ssum{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < TN; ++i) dc[q][i] = db[q][i] = floatx4{0, 0, 0, 0};

    const uint32_t pairs = hpg * a.nslice, per = (pairs + a.nsplit - 1) / a.nsplit;
    for (uint32_t v = sp * per; v < min(pairs, (sp + 1) * per); ++v) {
        const uint32_t h = g * hpg + v / a.nslice, sl = v % a.nslice, p0 = sl * GP, pn = min((uint32_t)GP, P - p0);
        const size_t row0 = ((size_t)b * L + t0) * a.H * P + (size_t)h * P + p0, hp = (size_t)a.H * P;
        const size_t slot = (((size_t)b * a.H + h) * a.nchunk + c) * P * N + (size_t)p0 * N;
        __syncthreads();
        load_tile<T, GP>(Xs, GXP, (const T*)a.X + row0, hp, tl, pn);
        load_tile<T, GP>(Ys, GXP, (const T*)a.dY + row0, hp, tl, pn);
        load_tile<float, NT>(Hs, NP, a.hst + slot, N, pn, N);
        load_tile<float, NT>(Gs, NP, a.gst + slot, N, pn, N);
        double tot = 0.0;
        if (w == 0) {
            const Steps st = chunk_steps<T>(a, b, h, t0, tl);
            tot = st.tot;
            if (lane < GQ) {
                Lc[lane] = st.lc;
                DT[lane] = st.dt;
                EL[lane] = (float)exp(st.lc);
                ER[lane] = (float)exp(st.tot - st.lc);
            }
        }
        __syncthreads();
        // S and M of this wave's tile; row and column sums of K
        floatx4 sd{0, 0, 0, 0};
        if (T0 >= J0)
            for (int k = 0; k < GP / 4; ++k)
                sd = mma4(Ys[(16 * T0 + li) * GXP + 4 * k + lq], Xs[(16 * J0 + li) * GXP + 4 * k + lq], sd);
        const int j = 16 * J0 + li;
        float col = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = 16 * T0 + 4 * lq + r;
            const float e = t >= j ? expf((float)(Lc[t] - Lc[j])) : 0.0f;
            const float m = cb[r] * e, kk = sd[r] * m;
            ssum[r] += sd[r] * e * DT[j];
            Ms[t * GXP + j] = m;
            const float row = group_sum<16>(kk * DT[j]);
            if (li == 0) RS[J0][t] = row;
            col += kk;
        }
        col += __shfl_xor(col, 16);
        col += __shfl_xor(col, 32);
        if (lq == 0) CS[T0][j] = col;
        // the parts that meet the states
        float vo[2][4] = {};
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const int n = 16 * (w + 4 * i) + li;
                floatx4 x{0, 0, 0, 0}, y{0, 0, 0, 0};
                for (int k = 0; k < GP / 4; ++k) {
                    x = mma4(Ys[(16 * q + li) * GXP + 4 * k + lq], Hs[(4 * k + lq) * NP + n], x);
                    y = mma4(Xs[(16 * q + li) * GXP + 4 * k + lq], Gs[(4 * k + lq) * NP + n], y);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = 16 * q + 4 * lq + r;
                    const float d = EL[t] * x[r];
                    dc[q][i][r] += d;
                    vo[q][r] += d * Cs[t * NP + n];
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
        for (int k = 0; k < NT / 4; ++k)
            dx = mma4(Bs[(16 * T0 + li) * NP + 4 * k + lq], Gs[(16 * J0 + li) * NP + 4 * k + lq], dx);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = 16 * T0 + 4 * lq + r;
            dx[r] *= ER[t];
            const float u = group_sum<16>(dx[r] * Xs[t * GXP + 16 * J0 + li]);
            if (li == 0) UO[J0][t] = u;
        }
        float gh = 0.0f, yx = 0.0f;
        for (int i = tid; i < GP * NT; i += G_NT) gh += Hs[i / NT * NP + i % NT] * Gs[i / NT * NP + i % NT];
        for (int i = tid; i < GQ * GP; i += G_NT) yx += Xs[i / GP * GXP + i % GP] * Ys[i / GP * GXP + i % GP];
        gh = wave_sum(gh);
        yx = wave_sum(yx);
        if (lane == 0) {
            red[w][0] = gh;
            red[w][1] = yx;
        }
        __syncthreads();
        for (int k = 0; k < GQ / 4; ++k)
            dx = mma4(Ms[(4 * k + lq) * GXP + 16 * T0 + li], Ys[(4 * k + lq) * GXP + 16 * J0 + li], dx);
        const float D = a.D ? to_f(((const T*)a.D)[h]) : 0.0f;
        const uint32_t p = 16 * J0 + li;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t t = 16 * T0 + 4 * lq + r;
            if (t < tl && p < pn) ((T*)a.dX)[row0 + t * hp + p] = from_f<T>(fmaf(DT[t], dx[r], D * Ys[t * GXP + p]));
        }
        // a_t: pairs of a source before t and a sink from t on
        if (w == 0) {
            const int t = min(lane, GQ - 1);
            const float dt = lane < GQ ? DT[t] : 0.0f, uo = UO[0][t] + UO[1][t], cs = CS[0][t] + CS[1][t];
            float pre = lane < GQ ? dt * uo : 0.0f;
            const float own = pre;
            float suf = lane < GQ ? (VO[0][t] + VO[1][t]) + (VO[2][t] + VO[3][t]) + (RS[0][t] + RS[1][t]) - dt * cs : 0.0f;
#pragma unroll
            for (int d = 1; d < GQ; d <<= 1) {
                const float x = __shfl_up(pre, d), y = __shfl_down(suf, d);
                if (lane >= d) pre += x;
                if (lane + d < GQ) suf += y;
            }
            const float edge = (float)exp(tot) * ((red[0][0] + red[1][0]) + (red[2][0] + red[3][0]));
            const float da = edge + (pre - own) + suf;
            const float A = -expf(to_f(((const T*)a.A_log)[h]));
            if (lane < (int)tl) a.q[(((size_t)sl * a.batch + b) * a.H + h) * L + t0 + lane] = uo + cs + A * da;
            const float dA = wave_sum(dt * da);
            if (lane == 0) {
                float* o = a.part + ((((size_t)b * a.H + h) * a.nslice + sl) * a.nchunk + c) * 2;
                o[0] = A * dA;
                o[1] = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
            }
        }
    }
    // within the chunk: sum of S over the share's heads with B and C
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) Ms[(16 * T0 + 4 * lq + r) * GXP + 16 * J0 + li] = ssum[r];
    __syncthreads();
    const size_t base = (size_t)sp * a.batch * L * a.G * N;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const uint32_t n = 16 * (w + 4 * i) + li;
            for (int k = 0; k < GQ / 4; ++k) {
                dc[q][i] = mma4(Ms[(16 * q + li) * GXP + 4 * k + lq], Bs[(4 * k + lq) * NP + n], dc[q][i]);
                db[q][i] = mma4(Ms[(4 * k + lq) * GXP + 16 * q + li], Cs[(4 * k + lq) * NP + n], db[q][i]);
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
// Sums over shares, slices and chunks
// ---------------------------------------------------------------------------
// gradient of raw + bias from that of dt: the softplus' slope, 0 where the
// clamp holds
template <typename T> __device__ __forceinline__ float dt_slope(const SsdBwdArgs& a, uint32_t b, uint32_t t, uint32_t h) {
    const float v = to_f(((const T*)a.dt)[((size_t)b * a.L + t) * a.H + h]) + to_f(((const T*)a.dt_bias)[h]);
    const float sp = v > 20.0f ? v : log1pf(expf(v));
    return sp >= a.dt_min && sp <= a.dt_max ? 1.0f / (1.0f + expf(-v)) : 0.0f;
}
__device__ __forceinline__ float dt_grad(const SsdBwdArgs& a, uint32_t b, uint32_t t, uint32_t h) {
    float s = 0.0f;
    for (uint32_t i = 0; i < a.nslice; ++i) s += a.q[(((size_t)i * a.batch + b) * a.H + h) * a.L + t];
    return s;
}

template <typename T> __global__ __launch_bounds__(256) void ssd_bwd_rows_kernel(SsdBwdArgs a) {
    const size_t nb = (size_t)a.batch * a.L * a.G * a.N, nt = (size_t)a.batch * a.L * a.H;
    const size_t step = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < nb; i += step) {
        float x = 0.0f, y = 0.0f;
        for (uint32_t s = 0; s < a.nsplit; ++s) {
            x += a.bpart[s * nb + i];
            y += a.cpart[s * nb + i];
        }
        ((T*)a.dB)[i] = from_f<T>(x);
        ((T*)a.dC)[i] = from_f<T>(y);
    }
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < nt; i += step) {
        const uint32_t h = i % a.H, b = i / a.H / a.L, t = i / a.H % a.L;
        ((T*)a.d_dt)[i] = from_f<T>(dt_grad(a, b, t, h) * dt_slope<T>(a, b, t, h));
    }
}

// A head's sums over all tokens, in 64 bits: a block a head.
template <typename T> __global__ __launch_bounds__(256) void ssd_bwd_heads_kernel(SsdBwdArgs a) {
    __shared__ double red[3][256];
    const uint32_t h = blockIdx.x, tid = threadIdx.x;
    double s[3] = {0, 0, 0};
    for (size_t i = tid; i < (size_t)a.batch * a.L; i += 256) {
        const uint32_t b = i / a.L, t = i % a.L;
        s[0] += (double)(dt_grad(a, b, t, h) * dt_slope<T>(a, b, t, h));
    }
    const size_t np = (size_t)a.nslice * a.nchunk;
    for (size_t i = tid; i < a.batch * np; i += 256) {
        const float* o = a.part + (((size_t)(i / np) * a.H + h) * np + i % np) * 2;
        s[1] += (double)o[0];
        s[2] += (double)o[1];
    }
    for (int k = 0; k < 3; ++k) red[k][tid] = s[k];
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
        if ((int)tid < d)
            for (int k = 0; k < 3; ++k) red[k][tid] += red[k][tid + d];
        __syncthreads();
    }
    if (tid == 0) {
        ((T*)a.d_dt_bias)[h] = from_f<T>((float)red[0][0]);
        ((T*)a.dA_log)[h] = from_f<T>((float)red[1][0]);
        if (a.dD) ((T*)a.dD)[h] = from_f<T>((float)red[2][0]);
    }
}

template <typename F> hipError_t with_type(int act, F f) {
    if (act == LSSM_BF16) return f(bf16{});
    if (act == LSSM_F16) return f(f16{});
    return f(float{});
}

// The plan and the workspace: [h0 states][G1 states][dB parts][dC parts][q][head parts]
struct Plan {
    uint32_t nchunk, nslice, nsplit;
    size_t states, rows, q, part;      // floats of one of each
    size_t floats() const { return 2 * states + 2 * rows + q + part; }
};
Plan plan_of(uint32_t batch, const lssm_ssd_dims& d) {
    Plan p;
    p.nchunk = (d.L + GQ - 1) / GQ;
    p.nslice = (d.P + GP - 1) / GP;
    const uint32_t pairs = d.H / d.n_groups * p.nslice;
    // shares of a group's heads: two blocks a CU where there are that many
    const size_t blocks = std::max<size_t>(1, (size_t)p.nchunk * batch * d.n_groups);
    p.nsplit = (uint32_t)std::min<size_t>(pairs, (512 + blocks - 1) / blocks);
    p.nsplit = (pairs + (pairs + p.nsplit - 1) / p.nsplit - 1) / ((pairs + p.nsplit - 1) / p.nsplit);
    p.states = (size_t)batch * d.H * p.nchunk * d.P * d.N;
    p.rows = (size_t)p.nsplit * batch * d.L * d.n_groups * d.N;
    p.q = (size_t)p.nslice * batch * d.H * d.L;
    p.part = (size_t)batch * d.H * p.nslice * p.nchunk * 2;
    return p;
}

template <typename T, int NT> void launch_generic(hipStream_t s, const SsdBwdArgs& a) {
    ssd_bwd_walk_kernel<T, NT><<<dim3(a.H * a.nslice, a.batch, 2), G_NT, 0, s>>>(a);
    if (a.nchunk)
        ssd_bwd_chunk_kernel<T, NT><<<dim3(a.nchunk * a.nsplit * a.G, a.batch), G_NT, 0, s>>>(a);
}

}  // namespace

size_t ssd_bwd_ws_bytes(uint32_t batch, const lssm_ssd_dims& d, int act) {
    (void)act;
    return plan_of(batch, d).floats() * sizeof(float);
}

hipError_t launch_ssd_bwd(hipStream_t s, SsdBwdArgs a, const lssm_ssd_dims& d, int act, void* ws) {
    const Plan p = plan_of(a.batch, d);
    a.nchunk = p.nchunk;
    a.nslice = p.nslice;
    a.nsplit = p.nsplit;
    a.hst = static_cast<float*>(ws);
    a.gst = a.hst + p.states;
    a.bpart = a.gst + p.states;
    a.cpart = a.bpart + p.rows;
    a.q = a.cpart + p.rows;
    a.part = a.q + p.q;
    return with_type(act, [&](auto z) {
        using T = decltype(z);
        if (a.batch) {
            if (a.N <= 64) launch_generic<T, 64>(s, a);
            else if (a.N <= 128) launch_generic<T, 128>(s, a);
            else launch_generic<T, 256>(s, a);
            const size_t n = (size_t)a.batch * a.L * std::max(a.G * a.N, a.H);
            if (n)
                ssd_bwd_rows_kernel<T><<<(uint32_t)std::min<size_t>((n + 255) / 256, 4096), 256, 0, s>>>(a);
        }
        ssd_bwd_heads_kernel<T><<<a.H, 256, 0, s>>>(a);
        return hipGetLastError();
    });
}

}  // namespace lssm
