// selective_scan.hip - selective state space scan: forward, backward, single step.
//
//   dt = softplus(delta + bias);  h_t = exp(dt A) h_{t-1} + dt B_t u_t;  y_t = C_t . h_t + D u_t;  out = y z sigmoid(z)
//   (per channel d a state of N numbers; B_t, C_t shared by the channels of a group; h := 0 before a step flagged as a reset)
//
// Layout.  A workgroup owns 64 consecutive channels of one group and walks along time in tiles of 16 steps; wave w owns states
// 4w .. 4w+3 of all 64 channels (lane = channel), so N = 16 is four waves.  What does not depend on the state index - softplus, the
// products dt u, the gate - is formed once per (step, channel) by whichever wave stages that row and goes through LDS; per (step,
// channel, state) there remain one multiply, one v_exp_f32, one multiply and two FMAs.  The sums over states (y, and in the backward
// the two sums behind du and ddelta) are joined through LDS, in a fixed order.
// The vector ALU bounds these kernels (v_exp_f32 takes four issue slots of the eight per state), the bytes come second.
#include "seq_common.hpp"

namespace {

constexpr int kTile = 16;              // steps per tile
constexpr int kLanes = 64;             // channels per workgroup

struct ScanArgs {
    const void *u, *delta, *z, *Bm, *Cm;
    const float *A, *Dskip, *bias, *s0;
    const int* lengths;
    const unsigned char* resets;
    long long ub, ut, db, dt, zb, zt, bb, bt, bg, cb, ct, cg, rb, rt;
    void* out;
    float *s1, *ckpt;
    int B, T, D, N, G, softplus;
    int Dg, nb, tiles;                 // channels per group, workgroups per group, tiles of T
};

struct ScanGradArgs {
    const void* dout;
    long long ob, ot;
    const float* ds1;
    void *du, *ddelta, *dz, *dB, *dC;
    float* ds0;
    float *param_partials, *bc_partials;
    int rows;                          // workgroups along the batch
};

// reset flags of the tile's steps as a wave-uniform bit mask
__device__ __forceinline__ unsigned reset_bits(const ScanArgs& a, int b, int t0, int nv, int lane) {
    if (!a.resets) return 0;
    const bool f = lane < nv && a.resets[b * a.rb + (t0 + lane) * a.rt] != 0;
    return (unsigned)__ballot(f);
}

__device__ __forceinline__ float time_step(const ScanArgs& a, float raw) { return a.softplus ? softplus(raw) : raw; }

template <typename T, int NG>
__global__ __launch_bounds__(kLanes* NG) void scan_fwd_kernel(ScanArgs a) {
    constexpr int kRows = kTile / NG, kStates = 4 * NG;
    __shared__ float sdt[kTile][kLanes], sdtu[kTile][kLanes], sy[NG][kTile][kLanes];
    __shared__ alignas(16) float sB[kTile][kStates], sC[kTile][kStates];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % a.nb, g = (blockIdx.x / a.nb) % a.G, b = blockIdx.x / (a.nb * a.G);
    const int ch = cb * kLanes + lane;
    const bool live = ch < a.Dg;
    const int d = g * a.Dg + (live ? ch : a.Dg - 1);
    const int len = seq_len(a.lengths, b, a.T);
    const T* u = (const T*)a.u + b * a.ub + d;
    const T* delta = (const T*)a.delta + b * a.db + d;
    const T* z = a.z ? (const T*)a.z + b * a.zb + d : nullptr;
    const T* Bm = (const T*)a.Bm + b * a.bb + g * a.bg;
    const T* Cm = (const T*)a.Cm + b * a.cb + g * a.cg;
    T* out = (T*)a.out + (long long)b * a.T * a.D + d;
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;

    float A2[4], h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = 4 * w + j;
        A2[j] = n < a.N ? a.A[(long long)d * a.N + n] * kLog2e : 0.0f;
        h[j] = n < a.N && a.s0 ? a.s0[((long long)b * a.D + d) * a.N + n] : 0.0f;
    }
    const int brow = threadIdx.x / kStates, bn = threadIdx.x % kStates;
    for (int t0 = 0; t0 < len; t0 += kTile) {
        const int nv = min(kTile, len - t0);
        if (a.ckpt && t0 && live)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (4 * w + j < a.N)
                    a.ckpt[(((long long)b * (a.tiles - 1) + t0 / kTile - 1) * a.D + d) * a.N + 4 * w + j] = h[j];
        float uu[kRows], zz[kRows];
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int r = w + k * NG, t = t0 + r;
            float dt = 0.0f;
            uu[k] = zz[k] = 0.0f;
            if (r < nv) {
                uu[k] = to_f32(u[t * a.ut]);
                dt = time_step(a, to_f32(delta[t * a.dt]) + bias);
                if (z) zz[k] = to_f32(z[t * a.zt]);
            }
            sdt[r][lane] = dt;
            sdtu[r][lane] = dt * uu[k];
        }
        const bool bl = brow < nv && bn < a.N;
        sB[brow][bn] = bl ? to_f32(Bm[(t0 + brow) * a.bt + bn]) : 0.0f;
        sC[brow][bn] = bl ? to_f32(Cm[(t0 + brow) * a.ct + bn]) : 0.0f;
        const unsigned cut = reset_bits(a, b, t0, nv, lane);
        __syncthreads();
#pragma unroll 4
        for (int r = 0; r < nv; r++) {
            if (cut >> r & 1) h[0] = h[1] = h[2] = h[3] = 0.0f;
            const float dt = sdt[r][lane], dtu = sdtu[r][lane];
            const float4 Bv = *(const float4*)&sB[r][4 * w], Cv = *(const float4*)&sC[r][4 * w];
            const float B4[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, C4[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
            float y = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                h[j] = __builtin_fmaf(exp2_hw(dt * A2[j]), h[j], dtu * B4[j]);
                y = __builtin_fmaf(C4[j], h[j], y);
            }
            sy[w][r][lane] = y;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int r = w + k * NG;
            float y = skip * uu[k];
#pragma unroll
            for (int v = 0; v < NG; v++) y += sy[v][r][lane];
            if (z) y *= zz[k] * sigmoid(zz[k]);
            if (r < nv && live) out[(long long)(t0 + r) * a.D] = from_f32<T>(y);
        }
    }
    if (live) {
        for (int t = len + w; t < a.T; t += NG) out[(long long)t * a.D] = from_f32<T>(0.0f);
        if (a.s1)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (4 * w + j < a.N) a.s1[((long long)b * a.D + d) * a.N + 4 * w + j] = h[j];
    }
}

// Sums of 8 registers over the 64 lanes, transposed on the way so that the number of live registers halves with every step (18
// instructions instead of 48): lane l returns the sum of v[order(l >> 3)].
__device__ __forceinline__ float sum_lanes8(const float* v, int lane) {
    float p[4], q[2];
#pragma unroll
    for (int i = 0; i < 4; i++) {       // lanes 0..31: v[2i], lanes 32..63: v[2i+1]
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), false, false);
        p[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {       // rows of 16: p[2i], p[2i+1], p[2i], p[2i+1]
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(p[2 * i]), __float_as_uint(p[2 * i + 1]), false, false);
        q[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    const bool up = lane & 8;
    const float mine = up ? q[1] : q[0], other = up ? q[0] : q[1];
    float r = mine + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(other), 0x128, 0xf, 0xf, true));   // row_ror:8
    r += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(r), 0x141, 0xf, 0xf, true));                   // row_half_mirror
    r += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(r), 0x4E, 0xf, 0xf, true));                    // quad_perm [2,3,0,1]
    r += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(r), 0xB1, 0xf, 0xf, true));                    // quad_perm [1,0,3,2]
    return r;
}
// index of the register whose sum the lanes 8g .. 8g+7 hold
__device__ __forceinline__ int sum_lanes8_order(int lane) {
    const int half = lane >> 5, odd = (lane >> 4) & 1, up = (lane >> 3) & 1;
    return 4 * up + 2 * odd + half;
}

// Reverse pass.  g_t = C_t dy_t + a_{t+1} g_{t+1} is the gradient of h_t; with q = g_t a_t h_{t-1}:
//   s1 = sum_n g B, s2 = sum_n q A:  du = dt s1 + D dy,  ddt = u s1 + s2;   dA += q dt;   dB = sum_d g dt u;   dC = sum_d dy h
// The states of a tile are run again from the state the forward left before it and kept, with the decays, in registers; tiles are
// walked backwards.  A workgroup takes every `rows`-th sequence, so that dA, dD and the bias gradient stay in registers meanwhile.
template <typename T, int NG, bool kResets>
__global__ __launch_bounds__(kLanes* NG) void scan_bwd_kernel(ScanArgs a, ScanGradArgs q) {
    constexpr int kRows = kTile / NG, kStates = 4 * NG;
    __shared__ float sdt[kTile][kLanes], sdtu[kTile][kLanes], sdy[kTile][kLanes];
    __shared__ float sy[NG][kTile][kLanes], ss1[NG][kTile][kLanes], ss2[NG][kTile][kLanes];
    __shared__ alignas(16) float sB[kTile][kStates], sC[kTile][kStates];
    __shared__ float sdB[kTile][kStates], sdC[kTile][kStates];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % a.nb, g = (blockIdx.x / a.nb) % a.G, row = blockIdx.x / (a.nb * a.G);
    const int ch = cb * kLanes + lane;
    const bool live = ch < a.Dg;
    const int d = g * a.Dg + (live ? ch : a.Dg - 1);
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;
    const int brow = threadIdx.x / kStates, bn = threadIdx.x % kStates;
    float A1[4], dA[4], dD = 0.0f, dbias = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = 4 * w + j;
        A1[j] = n < a.N ? a.A[(long long)d * a.N + n] : 0.0f;
        dA[j] = 0.0f;
    }
    for (int b = row; b < a.B; b += q.rows) {
        const int len = seq_len(a.lengths, b, a.T);
        const T* u = (const T*)a.u + b * a.ub + d;
        const T* delta = (const T*)a.delta + b * a.db + d;
        const T* z = a.z ? (const T*)a.z + b * a.zb + d : nullptr;
        const T* dout = (const T*)q.dout + b * q.ob + d;
        const T* Bm = (const T*)a.Bm + b * a.bb + g * a.bg;
        const T* Cm = (const T*)a.Cm + b * a.cb + g * a.cg;
        const long long o = (long long)b * a.T * a.D + d;
        float carry[4];                          // a_{t+1} g_{t+1}
#pragma unroll
        for (int j = 0; j < 4; j++)
            carry[j] = q.ds1 && live && 4 * w + j < a.N ? q.ds1[((long long)b * a.D + d) * a.N + 4 * w + j] : 0.0f;
        for (int tile = a.tiles - 1; tile >= 0; tile--) {
            const int t0 = tile * kTile, nv = max(0, min(kTile, len - t0)), nt = min(kTile, a.T - t0);
            float uu[kRows], dts[kRows], sg[kRows], zz[kRows], go[kRows];
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const int r = w + k * NG, t = t0 + r;
                uu[k] = dts[k] = sg[k] = zz[k] = go[k] = 0.0f;
                float dy = 0.0f;
                if (r < nv && live) {
                    uu[k] = to_f32(u[t * a.ut]);
                    const float raw = to_f32(delta[t * a.dt]) + bias;
                    dts[k] = time_step(a, raw);
                    sg[k] = a.softplus ? sigmoid(raw) : 1.0f;
                    go[k] = dy = to_f32(dout[t * q.ot]);
                    if (z) {
                        zz[k] = to_f32(z[t * a.zt]);
                        dy *= zz[k] * sigmoid(zz[k]);
                    }
                }
                sdt[r][lane] = dts[k];
                sdtu[r][lane] = dts[k] * uu[k];
                sdy[r][lane] = dy;
            }
            const bool bl = brow < nv && bn < a.N;
            sB[brow][bn] = bl ? to_f32(Bm[(t0 + brow) * a.bt + bn]) : 0.0f;
            sC[brow][bn] = bl ? to_f32(Cm[(t0 + brow) * a.ct + bn]) : 0.0f;
            const unsigned cut = reset_bits(a, b, t0, nv, lane);
            __syncthreads();
            if (nv) {
                float h[kTile + 1][4], e[kTile][4];
                const float* from = tile ? a.ckpt + ((long long)b * (a.tiles - 1) + tile - 1) * a.D * a.N
                                         : (a.s0 ? a.s0 + (long long)b * a.D * a.N : nullptr);
#pragma unroll
                for (int j = 0; j < 4; j++) h[0][j] = from && live && 4 * w + j < a.N ? from[(long long)d * a.N + 4 * w + j] : 0.0f;
#pragma unroll
                for (int r = 0; r < kTile; r++) {      // steps behind nv have dt = 0: decay 1, no input
                    const float dt = sdt[r][lane], dtu = sdtu[r][lane];
                    const float4 Bv = *(const float4*)&sB[r][4 * w], Cv = *(const float4*)&sC[r][4 * w];
                    const float B4[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, C4[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
                    float y = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const bool fresh = kResets && (cut >> r & 1);     // the state before is cleared, whatever it holds
                        e[r][j] = fresh ? 0.0f : exp2_hw(dt * (A1[j] * kLog2e));
                        h[r + 1][j] = __builtin_fmaf(e[r][j], fresh ? 0.0f : h[r][j], dtu * B4[j]);
                        y = __builtin_fmaf(C4[j], h[r + 1][j], y);
                    }
                    sy[w][r][lane] = y;
                }
                float sums = 0.0f;
#pragma unroll
                for (int r = kTile - 1; r >= 0; r--) {
                    const float dt = sdt[r][lane], dtu = sdtu[r][lane], dy = sdy[r][lane];
                    const float4 Bv = *(const float4*)&sB[r][4 * w], Cv = *(const float4*)&sC[r][4 * w];
                    const float B4[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, C4[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
                    float s1 = 0.0f, s2 = 0.0f, v[8];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float gr = __builtin_fmaf(C4[j], dy, carry[j]);
                        v[j] = gr * dtu;
                        v[4 + j] = dy * h[r + 1][j];
                        s1 = __builtin_fmaf(gr, B4[j], s1);
                        carry[j] = kResets && (cut >> r & 1) ? 0.0f : e[r][j] * gr;
                        const float qq = kResets && (cut >> r & 1) ? 0.0f : carry[j] * h[r][j];
                        s2 = __builtin_fmaf(qq, A1[j], s2);
                        dA[j] = __builtin_fmaf(qq, dt, dA[j]);
                    }
                    ss1[w][r][lane] = s1;
                    ss2[w][r][lane] = s2;
                    // lanes 8g + (r & 7) keep step r's sums; eight steps later all lanes have one to store
                    const float s = sum_lanes8(v, lane);
                    sums = (lane & 7) == (r & 7) ? s : sums;
                    if ((r & 7) == 0) {
                        const int i = sum_lanes8_order(lane), rr = r + (lane & 7);
                        (i < 4 ? sdB : sdC)[rr][4 * w + (i & 3)] = sums;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const int r = w + k * NG;
                float y = skip * uu[k], s1 = 0.0f, s2 = 0.0f;
                if (r < nv) {
#pragma unroll
                    for (int v = 0; v < NG; v++) y += sy[v][r][lane], s1 += ss1[v][r][lane], s2 += ss2[v][r][lane];
                }
                float dy = go[k], dzv = 0.0f;
                if (z) {
                    const float s = sigmoid(zz[k]);
                    dzv = go[k] * y * (s * (1.0f + zz[k] * (1.0f - s)));
                    dy *= zz[k] * s;
                }
                const float draw = (uu[k] * s1 + s2) * sg[k];
                if (r < nt && live) {
                    const long long at = o + (long long)(t0 + r) * a.D;
                    ((T*)q.du)[at] = from_f32<T>(__builtin_fmaf(dts[k], s1, skip * dy));
                    ((T*)q.ddelta)[at] = from_f32<T>(draw);
                    if (z) ((T*)q.dz)[at] = from_f32<T>(dzv);
                }
                dD = __builtin_fmaf(dy, uu[k], dD);
                dbias += draw;
            }
            if (brow < nt && bn < a.N) {
                const float vB = brow < nv ? sdB[brow][bn] : 0.0f, vC = brow < nv ? sdC[brow][bn] : 0.0f;
                const long long at = (((long long)b * a.T + t0 + brow) * a.G + g) * a.N + bn, n = (long long)a.B * a.T * a.G * a.N;
                if (q.bc_partials) {
                    q.bc_partials[(2 * cb) * n + at] = vB;
                    q.bc_partials[(2 * cb + 1) * n + at] = vC;
                } else {
                    ((T*)q.dB)[at] = from_f32<T>(vB);
                    ((T*)q.dC)[at] = from_f32<T>(vC);
                }
            }
        }
        if (q.ds0 && live)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (4 * w + j < a.N) q.ds0[((long long)b * a.D + d) * a.N + 4 * w + j] = carry[j];
    }
    // this workgroup's row of partial parameter gradients: [rows, D, N + 2]
    float* part = q.param_partials + ((long long)row * a.D + d) * (a.N + 2);
    __syncthreads();
    sdt[2 * w][lane] = dD, sdt[2 * w + 1][lane] = dbias;
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (4 * w + j < a.N) part[4 * w + j] = dA[j];
    if (w == 0) {
        float s = 0.0f, p = 0.0f;
#pragma unroll
        for (int v = 0; v < NG; v++) s += sdt[2 * v][lane], p += sdt[2 * v + 1][lane];
        part[a.N] = s;
        part[a.N + 1] = p;
    }
}

__global__ __launch_bounds__(256) void scan_params_kernel(const float* partials, int rows, int D, int N, float* dA, float* dD, float* dbias) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, n = (long long)D * (N + 2);
    if (i >= n) return;
    float s = 0.0f;
    for (int r = 0; r < rows; r++) s += partials[r * n + i];
    const int d = (int)(i / (N + 2)), k = (int)(i - (long long)d * (N + 2));
    if (k < N) dA[(long long)d * N + k] = s;
    else if (k == N) { if (dD) dD[d] = s; }
    else if (dbias) dbias[d] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void scan_bc_kernel(const float* partials, int nb, long long n, T* dB, T* dC) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * n) return;
    float s = 0.0f;
    for (int c = 0; c < nb; c++) s += partials[c * 2 * n + i];
    if (i < n) dB[i] = from_f32<T>(s);
    else dC[i - n] = from_f32<T>(s);
}

// One step: a channel's state is spread over L lanes, four numbers each, so that a wave moves 1 KB of states per access.
template <typename T, int L>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
    const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) / L;
    const int part = threadIdx.x % L;
    const bool live = item < (long long)a.B * a.D;
    const int b = live ? (int)(item / a.D) : 0, d = live ? (int)(item - (long long)b * a.D) : 0, g = d / a.Dg;
    const T* Bm = (const T*)a.Bm + b * a.bb + g * a.bg;
    const T* Cm = (const T*)a.Cm + b * a.cb + g * a.cg;
    const float uu = to_f32(((const T*)a.u)[b * a.ub + d]);
    const float dt = time_step(a, to_f32(((const T*)a.delta)[b * a.db + d]) + (a.bias ? a.bias[d] : 0.0f));
    const bool cut = a.resets && a.resets[b * a.rb];
    float y = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = 4 * part + j;
        if (n >= a.N) break;
        const long long at = ((long long)b * a.D + d) * a.N + n;
        float h = a.s0 && !cut ? a.s0[at] : 0.0f;
        h = __builtin_fmaf(exp2_hw(dt * (a.A[(long long)d * a.N + n] * kLog2e)), h, dt * uu * to_f32(Bm[n]));
        y = __builtin_fmaf(to_f32(Cm[n]), h, y);
        if (live) a.s1[at] = h;
    }
    if (L > 1) y += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(y), 0xB1, 0xf, 0xf, true));
    if (L > 2) y += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(y), 0x4E, 0xf, 0xf, true));
    if (L > 4) y += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(y), 0x141, 0xf, 0xf, true));
    if (!live || part) return;
    y = __builtin_fmaf(a.Dskip ? a.Dskip[d] : 0.0f, uu, y);
    if (a.z) {
        const float zz = to_f32(((const T*)a.z)[b * a.zb + d]);
        y *= zz * sigmoid(zz);
    }
    ((T*)a.out)[item] = from_f32<T>(y);
}

int tiles_of(int T) { return (T + kTile - 1) / kTile; }
int groups_of(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8; }
int channel_blocks(int D, int G) { return (D / G + kLanes - 1) / kLanes; }

// workgroups along the batch in the backward: a few per CU
int grad_rows(int B, int D, int G) {
    const int per = channel_blocks(D, G) * G, want = (2048 + per - 1) / per;
    return B < want ? B : want;
}

int check(const ag_scan_args* p) {
    if (!p || p->struct_size != sizeof(ag_scan_args) || !p->u_dev || !p->delta_dev || !p->Bm_dev || !p->Cm_dev || !p->A_dev)
        return AG_ERR_INVALID_ARG;
    if (p->B <= 0 || p->T <= 0 || p->D <= 0 || p->G <= 0 || p->N <= 0 || p->D % p->G) return AG_ERR_INVALID_ARG;
    if (p->N > 32 || p->dtype < AG_F32 || p->dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    if ((long long)p->B * p->G * channel_blocks(p->D, p->G) > 0x7fffffffLL) return AG_ERR_UNSUPPORTED;
    return AG_OK;
}

ScanArgs device_args(const ag_scan_args* p) {
    return ScanArgs{p->u_dev, p->delta_dev, p->z_dev, p->Bm_dev, p->Cm_dev, p->A_dev, p->Dskip_dev, p->delta_bias_dev, p->state_in_dev,
                    p->lengths_dev, p->resets_dev, p->u_sb, p->u_st, p->delta_sb, p->delta_st, p->z_sb, p->z_st, p->b_sb, p->b_st, p->b_sg,
                    p->c_sb, p->c_st, p->c_sg, p->r_sb, p->r_st, p->out_dev, p->state_out_dev, p->ckpt_dev, p->B, p->T, p->D, p->N, p->G,
                    p->softplus, p->D / p->G, channel_blocks(p->D, p->G), tiles_of(p->T)};
}

}  // namespace

#define AG_FOR_STATES(N_, CALL)                                    \
    do {                                                           \
        switch (groups_of(N_)) {                                   \
            case 1: { constexpr int NG = 1; CALL; } break;         \
            case 2: { constexpr int NG = 2; CALL; } break;         \
            case 4: { constexpr int NG = 4; CALL; } break;         \
            default: { constexpr int NG = 8; CALL; } break;        \
        }                                                          \
    } while (0)

extern "C" long long ag_selective_scan_ckpt_floats(int B, int T, int D, int N) {
    if (B <= 0 || T <= 0 || D <= 0 || N <= 0) return 0;
    return (long long)B * (tiles_of(T) - 1) * D * N;
}

extern "C" long long ag_selective_scan_workspace_bytes(int B, int T, int D, int N, int G, int backward) {
    if (B <= 0 || T <= 0 || D <= 0 || N <= 0 || G <= 0 || D % G || !backward) return 0;
    const int nb = channel_blocks(D, G);
    const long long params = (long long)grad_rows(B, D, G) * D * (N + 2);
    const long long bc = nb > 1 ? 2LL * nb * B * T * G * N : 0;
    return (params + bc) * (long long)sizeof(float);
}

extern "C" int ag_selective_scan_fwd(const ag_scan_args* p, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!p->out_dev) return AG_ERR_INVALID_ARG;
    const ScanArgs a = device_args(p);
    const dim3 grid((unsigned)((long long)a.B * a.G * a.nb));
    AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_fwd_kernel<T, NG>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a)));
    return seq_status();
}

extern "C" int ag_selective_scan_bwd(const ag_scan_args* p, const ag_scan_grads* s, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!s || s->struct_size != sizeof(ag_scan_grads) || !s->dout_dev || !s->du_dev || !s->ddelta_dev || !s->dBm_dev || !s->dCm_dev ||
        !s->dA_dev || !s->workspace_dev || (p->z_dev != nullptr) != (s->dz_dev != nullptr) || (p->T > kTile && !p->ckpt_dev))
        return AG_ERR_INVALID_ARG;
    if (s->workspace_bytes < ag_selective_scan_workspace_bytes(p->B, p->T, p->D, p->N, p->G, 1)) return AG_ERR_INVALID_ARG;
    const ScanArgs a = device_args(p);
    const int rows = grad_rows(a.B, a.D, a.G);
    float* params = (float*)s->workspace_dev;
    float* bc = a.nb > 1 ? params + (long long)rows * a.D * (a.N + 2) : nullptr;
    const ScanGradArgs q{s->dout_dev, s->dout_sb, s->dout_st, s->dstate_out_dev, s->du_dev, s->ddelta_dev, s->dz_dev, s->dBm_dev, s->dCm_dev,
                         s->dstate_in_dev, params, bc, rows};
    const dim3 grid((unsigned)((long long)rows * a.G * a.nb));
    if (a.resets)
        AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_bwd_kernel<T, NG, true>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a, q)));
    else
        AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_bwd_kernel<T, NG, false>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a, q)));
    const long long np = (long long)a.D * (a.N + 2);
    hipLaunchKernelGGL(scan_params_kernel, dim3((unsigned)((np + 255) / 256)), dim3(256), 0, (hipStream_t)stream, params, rows, a.D, a.N,
                       s->dA_dev, s->dDskip_dev, s->ddelta_bias_dev);
    if (bc) {
        const long long n = (long long)a.B * a.T * a.G * a.N;
        AG_FOR_DTYPE(p->dtype, hipLaunchKernelGGL((scan_bc_kernel<T>), dim3((unsigned)((2 * n + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                                                  bc, a.nb, n, (T*)s->dBm_dev, (T*)s->dCm_dev));
    }
    return seq_status();
}

extern "C" int ag_selective_scan_step(const ag_scan_args* p, void* stream) {
    if (const int rc = check(p)) return rc;
    if (p->T != 1 || !p->out_dev || !p->state_out_dev) return AG_ERR_INVALID_ARG;
    const ScanArgs a = device_args(p);
    const int lanes = groups_of(p->N);
    const long long blocks = ((long long)a.B * a.D * lanes + 255) / 256;
    if (blocks > 0x7fffffffLL) return AG_ERR_UNSUPPORTED;
    AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_step_kernel<T, NG>), dim3((unsigned)blocks), dim3(256), 0,
                                                                  (hipStream_t)stream, a)));
    return seq_status();
}
