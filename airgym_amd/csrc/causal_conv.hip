// causal_conv.hip - short causal depthwise convolution over padded sequences with episode resets: forward, backward, single step.
//
//   p[t] = bias + sum_k w[k] x[t-W+1+k]   (taps before the last reset are zero, before step 0 they are the state's)
//   y[t] = p sigmoid(p)  or  p
//
// One thread owns VEC neighbouring channels over a run of consecutive steps and carries the last W-1 inputs in registers, so that every
// input is read once per run plus W-1 steps of halo.  A workgroup is lx threads along the channels by ly runs.  Memory bounds it: the
// arithmetic is about 20 issue slots per element (half of them the sigmoid) for 4 to 8 bytes.  Hence accesses of 16 bytes where the
// channels divide (4 bytes or single channels where not), four steps' loads at a time, and runs short enough to have many in flight.
// At 4096 x 24 x 256, W = 4, float32, with resets: forward 37 us = 5.4 TB/s; backward 74 us = 4.1 TB/s, its vector pipe busy for half of
// the time, where 205 registers leave two waves per SIMD (three, by channels two at a time, took longer).
// The outputs are left to the caches: marked as used once the forward alone takes 34 us, but with the kernel that reads y 78 instead of 65.
#include "seq_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;              // steps whose loads are issued together

struct ConvArgs {
    const void* x; const float* w; const float* bias; const void* s0; const int* lengths; const unsigned char* resets;
    void* y; void* s1;
    long long xb, xt, rb, rt;
    int B, T, D, silu;
    int run, runs;                     // steps per thread, runs per sequence
    int lx, ly, nx;                    // threads along channels and along runs in a workgroup, workgroups along channels
};

struct ConvGradArgs {
    const void *dy, *ds1; void* dx; void* ds0; float* partials;
    long long dyb, dyt;
    int groups;                        // workgroups along the runs = rows of partial parameter gradients
};

// the W-1 inputs before step t0 as the convolution sees them there: the state's before step 0, zero from the last reset backwards, and
// zero behind the sequence's end, whatever stands there
template <typename T, int W, int VEC>
__device__ __forceinline__ void load_window(const ConvArgs& a, int b, int t0, int len, int d, float (*win)[VEC]) {
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        const int t = t0 - (W - 1) + j;
        const bool there = t < 0 ? a.s0 != nullptr : t < len;
        Vec<T, VEC> c;
        if (t >= 0 && there) {
            c = load_vec<T, VEC>((const T*)a.x + (b * a.xb + t * a.xt + d));
            if (a.resets && a.resets[b * a.rb + t * a.rt])
#pragma unroll
                for (int i = 0; i < j; i++)
#pragma unroll
                    for (int v = 0; v < VEC; v++) win[i][v] = 0.0f;
        } else if (there) c = load_vec<T, VEC>((const T*)a.s0 + (((long long)b * (W - 1) + (t + W - 1)) * a.D + d));
#pragma unroll
        for (int v = 0; v < VEC; v++) win[j][v] = there ? c.at(v) : 0.0f;
    }
}

template <typename T, int W, int VEC>
__device__ __forceinline__ void load_taps(const ConvArgs& a, int d, float (*w)[VEC], float* bias) {
#pragma unroll
    for (int v = 0; v < VEC; v++) {
#pragma unroll
        for (int k = 0; k < W; k++) w[k][v] = a.w[(long long)(d + v) * W + k];
        bias[v] = a.bias ? a.bias[d + v] : 0.0f;
    }
}

template <typename T, int W, int VEC>
__global__ __launch_bounds__(kThreads) void conv_fwd_kernel(ConvArgs a) {
    const int tx = threadIdx.x % a.lx, ty = threadIdx.x / a.lx;
    const int d = ((int)(blockIdx.x % a.nx) * a.lx + tx) * VEC;
    const long long row = (long long)(blockIdx.x / a.nx) * a.ly + ty;           // (b, run)
    if (ty >= a.ly || d >= a.D || row >= (long long)a.B * a.runs) return;
    const int b = (int)(row / a.runs), t0 = (int)(row - (long long)b * a.runs) * a.run;
    const int len = seq_len(a.lengths, b, a.T);
    const int t1 = min(t0 + a.run, a.T), tv = min(t1, len);
    const T* x = (const T*)a.x + (b * a.xb + d);
    T* y = (T*)a.y + ((long long)b * a.T * a.D + d);
    float w[W][VEC], bias[VEC], win[W][VEC];
    load_taps<T, W, VEC>(a, d, w, bias);
    if (t0 < tv || (len == 0 && t0 == 0)) load_window<T, W, VEC>(a, b, min(t0, len), len, d, win);
    auto step = [&](int t, const Vec<T, VEC>& c, unsigned char cut) __attribute__((always_inline)) {
        float p[VEC];
        if (a.resets)
#pragma unroll
            for (int j = 0; j < W - 1; j++)
#pragma unroll
                for (int v = 0; v < VEC; v++) win[j][v] = cut ? 0.0f : win[j][v];
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            win[W - 1][v] = c.at(v);
            p[v] = bias[v];
#pragma unroll
            for (int k = 0; k < W; k++) p[v] = __builtin_fmaf(w[k][v], win[k][v], p[v]);
        }
        if (a.silu)
#pragma unroll
            for (int v = 0; v < VEC; v++) p[v] *= sigmoid(p[v]);
        Vec<T, VEC> o;
        o.set(p);
        store_vec<T, VEC>(y + (long long)t * a.D, o);
#pragma unroll
        for (int j = 0; j < W - 1; j++)
#pragma unroll
            for (int v = 0; v < VEC; v++) win[j][v] = win[j + 1][v];
    };
    const unsigned char* flags = a.resets ? a.resets + b * a.rb : nullptr;
    int t = t0;
    for (; t + kAhead <= tv; t += kAhead) {
        Vec<T, VEC> c[kAhead];
        unsigned char cut[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            c[i] = load_vec<T, VEC>(x + (t + i) * a.xt);
            cut[i] = flags ? flags[(t + i) * a.rt] : 0;
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) step(t + i, c[i], cut[i]);
    }
    for (; t < tv; t++) step(t, load_vec<T, VEC>(x + t * a.xt), flags ? flags[t * a.rt] : 0);
    const float none[VEC] = {};
    Vec<T, VEC> zero;
    zero.set(none);
    for (t = max(t0, tv); t < t1; t++) store_vec<T, VEC>(y + (long long)t * a.D, zero);
    // the run that holds the last step (the first run of an empty sequence) leaves the state behind
    if (a.s1 && (len == 0 ? t0 == 0 : (t0 < len && len <= t0 + a.run))) {
        T* s1 = (T*)a.s1 + ((long long)b * (W - 1) * a.D + d);
#pragma unroll
        for (int j = 0; j < W - 1; j++) {
            Vec<T, VEC> o;
            o.set(win[j]);
            store_vec<T, VEC>(s1 + (long long)j * a.D, o);
        }
    }
}

// dp[t] = dy[t] act'(p[t]);  dx[t] = sum_k w[k] dp[t+W-1-k], the later step not behind a reset after t.  The thread walks on W-1
// steps past its run for the contributions of later steps; those steps' own parameter gradients belong to the next run.  A workgroup
// takes every `groups`-th block of runs, and adds up its own runs' parameter gradients.
template <typename T, int W, int VEC>
__global__ __launch_bounds__(kThreads) void conv_bwd_kernel(ConvArgs a, ConvGradArgs g) {
    __shared__ float sums[kThreads];
    const int tx = threadIdx.x % a.lx, ty = threadIdx.x / a.lx;
    const int dx0 = ((int)(blockIdx.x % a.nx) * a.lx + tx) * VEC, group = blockIdx.x / a.nx;
    const bool live = ty < a.ly && dx0 < a.D;
    const int d = live ? dx0 : 0;
    float w[W][VEC], bias[VEC], dw[W + 1][VEC];
    load_taps<T, W, VEC>(a, d, w, bias);
#pragma unroll
    for (int k = 0; k <= W; k++)
#pragma unroll
        for (int v = 0; v < VEC; v++) dw[k][v] = 0.0f;
    const long long rows = (long long)a.B * a.runs;
    if (live)
        for (long long row = (long long)group * a.ly + ty; row < rows; row += (long long)g.groups * a.ly) {
            const int b = (int)(row / a.runs), t0 = (int)(row - (long long)b * a.runs) * a.run, t1 = min(t0 + a.run, a.T);
            const int len = seq_len(a.lengths, b, a.T);
            const T* x = (const T*)a.x + (b * a.xb + d);
            const T* dy = (const T*)g.dy + (b * g.dyb + d);
            // the group's rows; the gradient written at step t is that of step t-W+1
            const T *px = x + t0 * a.xt, *pg = dy + t0 * g.dyt;
            T* dx = (T*)g.dx + (((long long)b * a.T + t0 - (W - 1)) * a.D + d);
            const unsigned char* flags = a.resets ? a.resets + (b * a.rb + t0 * a.rt) : nullptr;
            float win[W][VEC], acc[W][VEC];        // inputs and their gradients, oldest first
#pragma unroll
            for (int j = 0; j < W; j++)
#pragma unroll
                for (int v = 0; v < VEC; v++) acc[j][v] = 0.0f;
            load_window<T, W, VEC>(a, b, t0, len, d, win);
            const int some = min(len, t1 + W - 1);         // steps from here on have x = dy = 0: they add nothing
            int alive = W;                                 // taps that reach back over no reset since the run's start
            for (int t = t0; t < t1 + W - 1; t += kAhead) {
                Vec<T, VEC> cx[kAhead], cg[kAhead];
                unsigned char cut[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    const float none[VEC] = {};
                    cut[i] = 0;
                    if (t + i < some) {
                        cx[i] = load_vec<T, VEC>(px + i * a.xt);
                        cg[i] = load_vec<T, VEC>(pg + i * g.dyt);
                        if (flags) cut[i] = flags[i * a.rt];
                    } else cx[i].set(none), cg[i].set(none);
                }
                px += kAhead * a.xt, pg += kAhead * g.dyt;
                if (flags) flags += kAhead * a.rt;
                // No branch changes a window from here on: each would cost the copies that join its two sides.
#pragma unroll
                for (int i = 0; i < kAhead; i++) {
                    const int ti = t + i;
                    float dp[VEC], mine[VEC];
                    if (a.resets) {
                        alive = cut[i] ? 1 : alive;
#pragma unroll
                        for (int j = 0; j < W - 1; j++)
#pragma unroll
                            for (int v = 0; v < VEC; v++) win[j][v] = cut[i] ? 0.0f : win[j][v];
                    }
#pragma unroll
                    for (int v = 0; v < VEC; v++) win[W - 1][v] = cx[i].at(v), dp[v] = cg[i].at(v);
                    if (a.silu)
#pragma unroll
                        for (int v = 0; v < VEC; v++) {
                            float p = bias[v];
#pragma unroll
                            for (int k = 0; k < W; k++) p = __builtin_fmaf(w[k][v], win[k][v], p);
                            const float s = sigmoid(p);
                            dp[v] *= s * __builtin_fmaf(p, 1.0f - s, 1.0f);
                        }
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        mine[v] = ti < t1 ? dp[v] : 0.0f;
                        dw[W][v] += mine[v];
#pragma unroll
                        for (int k = 0; k < W; k++) dw[k][v] = __builtin_fmaf(mine[v], win[k][v], dw[k][v]);
                    }
                    if (a.resets) {
#pragma unroll
                        for (int k = 0; k < W; k++)
#pragma unroll
                            for (int v = 0; v < VEC; v++) acc[k][v] = __builtin_fmaf(w[k][v], k >= W - alive ? dp[v] : 0.0f, acc[k][v]);
                    } else {
#pragma unroll
                        for (int k = 0; k < W; k++)
#pragma unroll
                            for (int v = 0; v < VEC; v++) acc[k][v] = __builtin_fmaf(w[k][v], dp[v], acc[k][v]);
                    }
                    alive = ti < len ? min(alive + 1, W) : alive;
                    const int done = ti - (W - 1);         // this input has met every step that reads it
                    if (g.ds1 && ti >= len && done < len && len - 1 - done < alive - 1 && ti - len < W - 1) {
                        // ... and is part of the state left behind
                        const auto c = load_vec<T, VEC>((const T*)g.ds1 + (((long long)b * (W - 1) + (ti - len)) * a.D + d));
#pragma unroll
                        for (int v = 0; v < VEC; v++) acc[0][v] += c.at(v);
                    }
                    Vec<T, VEC> o;
                    o.set(acc[0]);
                    if (done >= t0) {
                        if (done < t1) store_vec<T, VEC>(dx + (long long)i * a.D, o);
                    } else if (t0 == 0 && g.ds0) store_vec<T, VEC>((T*)g.ds0 + (((long long)b * (W - 1) + ti) * a.D + d), o);
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
#pragma unroll
                        for (int j = 0; j < W - 1; j++) win[j][v] = win[j + 1][v], acc[j][v] = acc[j + 1][v];
                        acc[W - 1][v] = 0.0f;
                    }
                }
                dx += (long long)kAhead * a.D;
            }
        }
    // the workgroup's runs added up in order; one row of partial gradients [groups, D, W + 1]
    float* out = g.partials + ((long long)group * a.D + d) * (W + 1);
#pragma unroll
    for (int k = 0; k <= W; k++)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            if (a.ly > 1) {
                __syncthreads();
                sums[threadIdx.x] = dw[k][v];
                __syncthreads();
            }
            if (live && ty == 0) {
                float s = dw[k][v];
                for (int j = 1; j < a.ly; j++) s += sums[j * a.lx + tx];
                out[v * (W + 1) + k] = s;
            }
        }
}

struct ConvParams {
    float *dw, *db;
    int W;
    __device__ __forceinline__ void operator()(long long i, float s) const {
        const long long d = i / (W + 1);
        const int k = (int)(i - d * (W + 1));
        if (k < W) dw[d * W + k] = s;
        else if (db) db[d] = s;
    }
};

// One step: the state's rows are read, moved on by one and written back where they were.  Its bytes bound it (16384 x 2048, W = 4,
// float32: 6.0 TB/s, the second-level caches included; bfloat16 5.2 TB/s).
template <typename T, int W, int VEC, bool kOnce>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(const T* x, long long xb, T* state, const float* weight, const float* bias,
                                                            const unsigned char* resets, T* y, int B, int D, int silu) {
    const unsigned item = blockIdx.x * kThreads + threadIdx.x, dv = D / VEC, b = item / dv;      // B D < 2^31
    const int d = (int)(item - b * dv) * VEC;
    if (b >= (unsigned)B) return;
    T* s = state + ((long long)b * (W - 1) * D + d);
    const bool cut = resets && resets[b];
    const float none[VEC] = {};
    Vec<T, VEC> win[W];
#pragma unroll
    for (int j = 0; j < W - 1; j++) win[j] = load_vec<T, VEC, kOnce>(s + (long long)j * D);
    win[W - 1] = load_vec<T, VEC>(x + (b * xb + d));
    if (cut)
#pragma unroll
        for (int j = 0; j < W - 1; j++) win[j].set(none);
    float p[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        p[v] = bias ? bias[d + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) p[v] = __builtin_fmaf(weight[(long long)(d + v) * W + k], win[k].at(v), p[v]);
        if (silu) p[v] *= sigmoid(p[v]);
    }
    Vec<T, VEC> o;
    o.set(p);
    store_vec<T, VEC>(y + ((long long)b * D + d), o);
#pragma unroll
    for (int j = 0; j < W - 1; j++) store_vec<T, VEC, kOnce>(s + (long long)j * D, win[j + 1]);
}

// How the work is laid out, from sizes alone: channels per thread, threads along the channels, steps per run.
struct Plan { int vec, lx, ly, nx, run, runs; };
Plan plan_of(long long B, int T, int D, int wide) {
    Plan p;
    // what one access should hold (16 bytes in the forward); channels that do not divide move two or one
    p.vec = D % wide == 0 ? wide : D % 2 == 0 ? 2 : 1;
    const int dv = D / p.vec;
    p.lx = dv < kThreads ? dv : kThreads;
    p.ly = kThreads / p.lx;
    p.nx = (dv + p.lx - 1) / p.lx;
    // whole sequences per thread if that makes 4096 waves (16 per CU) or sequences are short; else runs of 16 steps and more
    const long long threads = B * dv;
    long long runs = (262144 + threads - 1) / threads;
    long long run = (T + runs - 1) / runs;
    run = (run + kAhead - 1) / kAhead * kAhead;
    p.run = (int)(run < 16 ? 16 : run);
    p.runs = (T + p.run - 1) / p.run;
    return p;
}

constexpr int wide_fwd(int size) { return 16 / size; }
// the backward holds 4 W + 1 rows of VEC in registers: four channels up to five taps, then two (W = 8 at 64 x 1000 x 512: 158 us with two,
// 194 with four)
constexpr int wide_bwd(int W) { return W <= 5 ? 4 : 2; }

// workgroups along the runs in the backward, each with one row of partial gradients
int grad_groups(const Plan& p, long long B) {
    const long long blocks = (B * p.runs + p.ly - 1) / p.ly, want = (1024 + p.nx - 1) / p.nx;
    return (int)(blocks < want ? blocks : want);
}

int check(const ag_conv_args* p) {
    if (!p || p->struct_size != sizeof(ag_conv_args) || !p->x_dev || !p->weight_dev) return AG_ERR_INVALID_ARG;
    if (p->B <= 0 || p->T <= 0 || p->D <= 0) return AG_ERR_INVALID_ARG;
    if (p->W < 2 || p->W > 8 || p->dtype < AG_F32 || p->dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    if (p->T > kMaxSteps) return AG_ERR_UNSUPPORTED;
    return AG_OK;
}

ConvArgs device_args(const ag_conv_args* p, const Plan& l) {
    return ConvArgs{p->x_dev, p->weight_dev, p->bias_dev, p->state_in_dev, p->lengths_dev, p->resets_dev, p->y_dev, p->state_out_dev,
                    p->x_sb, p->x_st, p->r_sb, p->r_st, p->B, p->T, p->D, p->silu, l.run, l.runs, l.lx, l.ly, l.nx};
}

}  // namespace

#define AG_FOR_TAPS(W_, CALL)                                            \
    do {                                                                 \
        switch (W_) {                                                    \
            case 2: { constexpr int W = 2; CALL; } break;                \
            case 3: { constexpr int W = 3; CALL; } break;                \
            case 4: { constexpr int W = 4; CALL; } break;                \
            case 5: { constexpr int W = 5; CALL; } break;                \
            case 6: { constexpr int W = 6; CALL; } break;                \
            case 7: { constexpr int W = 7; CALL; } break;                \
            case 8: { constexpr int W = 8; CALL; } break;                \
            default: return AG_ERR_UNSUPPORTED;                          \
        }                                                                \
    } while (0)

// run CALL with VEC bound to the plan's channels per thread
#define AG_FOR_VEC(vec, WIDE, CALL)                            \
    do {                                                       \
        if (vec == WIDE) { constexpr int VEC = WIDE; CALL; }   \
        else if (vec == 2) { constexpr int VEC = 2; CALL; }    \
        else { constexpr int VEC = 1; CALL; }                  \
    } while (0)

extern "C" int ag_causal_conv_fwd(const ag_conv_args* p, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!p->y_dev) return AG_ERR_INVALID_ARG;
    const int size = p->dtype == AG_F32 ? 4 : 2;
    const Plan l = plan_of(p->B, p->T, p->D, wide_fwd(size));
    const ConvArgs a = device_args(p, l);
    const long long blocks = ((long long)a.B * a.runs + l.ly - 1) / l.ly * l.nx;
    if (blocks > kMaxThreads / kThreads) return AG_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks);
    AG_FOR_DTYPE(p->dtype, AG_FOR_TAPS(p->W, AG_FOR_VEC(l.vec, wide_fwd(sizeof(T)), hipLaunchKernelGGL((conv_fwd_kernel<T, W, VEC>), grid,
                                                                                     dim3(kThreads), 0, (hipStream_t)stream, a))));
    return seq_status();
}

extern "C" long long ag_causal_conv_workspace_bytes(int B, int T, int D, int W, int dtype) {
    if (B <= 0 || T <= 0 || D <= 0 || W < 2 || W > 8 || dtype < AG_F32 || dtype > AG_F16) return 0;
    return (long long)grad_groups(plan_of(B, T, D, wide_bwd(W)), B) * D * (W + 1) * (long long)sizeof(float);
}

extern "C" int ag_causal_conv_bwd(const ag_conv_args* p, const ag_conv_grads* q, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!q || q->struct_size != sizeof(ag_conv_grads) || !q->dy_dev || !q->dx_dev || !q->dweight_dev || !q->workspace_dev)
        return AG_ERR_INVALID_ARG;
    if (q->workspace_bytes < ag_causal_conv_workspace_bytes(p->B, p->T, p->D, p->W, p->dtype)) return AG_ERR_INVALID_ARG;
    const Plan l = plan_of(p->B, p->T, p->D, wide_bwd(p->W));
    const ConvArgs a = device_args(p, l);
    const ConvGradArgs g{q->dy_dev, q->dstate_out_dev, q->dx_dev, q->dstate_dev, (float*)q->workspace_dev, q->dy_sb, q->dy_st,
                         grad_groups(l, a.B)};
    const dim3 grid((unsigned)(g.groups * l.nx));
    AG_FOR_DTYPE(p->dtype, AG_FOR_TAPS(p->W, AG_FOR_VEC(l.vec, wide_bwd(W), hipLaunchKernelGGL((conv_bwd_kernel<T, W, VEC>), grid,
                                                                                     dim3(kThreads), 0, (hipStream_t)stream, a, g))));
    launch_sum_rows(g.partials, g.groups, (long long)a.D * (p->W + 1), ConvParams{q->dweight_dev, q->dbias_dev, p->W}, stream);
    return seq_status();
}

extern "C" int ag_causal_conv_step(const void* x, long long x_sb, void* state, const float* weight, const float* bias,
                                   const unsigned char* resets, void* y, int dtype, int B, int D, int W_, int silu, void* stream) {
    if (!x || !state || !weight || !y || B <= 0 || D <= 0) return AG_ERR_INVALID_ARG;
    if (W_ < 2 || W_ > 8 || dtype < AG_F32 || dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    if ((long long)B * D > 0x7fffffffLL) return AG_ERR_UNSUPPORTED;
    // a dword per access: one float32 channel per thread, two of the 16-bit types where they divide.  Four are slower (16384 x 2048, W = 4:
    // float32 179, 191 and 199 us with 1, 2 and 4 channels; bfloat16 120, 103, 123 and 188 us with 1, 2, 4 and 8, 4.65, 4.05, 4.39 and
    // 5.16 us at 4096 x 256): the weights of a thread's channels are that many more gathered loads in front of the arithmetic.
    const int vec = dtype != AG_F32 && D % 2 == 0 ? 2 : 1;
    const unsigned blocks = (unsigned)(((long long)B * (D / vec) + kThreads - 1) / kThreads);
    // From half of the last-level cache on the states are marked as used once: plain and marked, in us, one batch moved on alone and three in turn,
    // at D = 2048, W = 4: float32 48 MiB 20.3, 23.1 and 20.2, 23.3; 127 MiB 49.6, 55.7 and 58.8, 55.7; 384 MiB 178, 162 and 178, 166; bfloat16 48 MiB
    // 23.3, 25.3 and 23.2, 25.6; 192 MiB 101, 88 and 103, 88.  (Between 60 and 128 MiB three in turn gain as well, one alone loses.)
    const bool once = (long long)B * D * (W_ - 1) * (dtype == AG_F32 ? 4 : 2) >= kCached;
#define AG_STEP(VEC, ONCE)                                                                                                         \
    AG_FOR_DTYPE(dtype, AG_FOR_TAPS(W_, hipLaunchKernelGGL((conv_step_kernel<T, W, VEC, ONCE>), dim3(blocks), dim3(kThreads), 0,     \
                                                           (hipStream_t)stream, (const T*)x, x_sb, (T*)state, weight, bias, resets, \
                                                           (T*)y, B, D, silu)))
    if (vec == 2 && once) AG_STEP(4 / sizeof(T), true);
    else if (vec == 2) AG_STEP(4 / sizeof(T), false);
    else if (once) AG_STEP(1, true);
    else AG_STEP(1, false);
#undef AG_STEP
    return seq_status();
}
