// causal_conv.hip - short causal depthwise convolution over padded sequences with episode resets: forward, backward, single step.
//
//   p[t] = bias + sum_k w[k] x[t-W+1+k]   (taps before the last reset are zero, before step 0 they are the state's)
//   y[t] = p sigmoid(p)  or  p
//
// One thread owns a channel over a run of consecutive steps and carries the last W-1 inputs in registers, so that every input is
// read once per run plus W-1 steps of halo.  Neighbouring lanes hold neighbouring channels.
#include "seq_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 32;               // steps per thread

struct ConvArgs {
    const void* x; const float* w; const float* bias; const void* s0; const int* lengths; const unsigned char* resets;
    void* y; void* s1;
    long long xb, xt, rb, rt;
    int B, T, D, silu, runs;
};

struct ConvGradArgs {
    const void *dy, *ds1; void* dx; void* ds0; float* partials;
    long long dyb, dyt;
    int rows;
};

// input at step t of sequence b; the state's before step 0
template <typename T, int W>
__device__ __forceinline__ float input_at(const ConvArgs& a, int b, int t, int d) {
    if (t >= 0) return to_f32(((const T*)a.x)[b * a.xb + t * a.xt + d]);
    return a.s0 ? to_f32(((const T*)a.s0)[((long long)b * (W - 1) + (t + W - 1)) * a.D + d]) : 0.0f;
}

// the W-1 inputs before step t0 as the convolution sees them there: zero from the last reset in the halo backwards
template <typename T, int W>
__device__ __forceinline__ void load_window(const ConvArgs& a, int b, int t0, int d, float* win) {
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        const int t = t0 - (W - 1) + j;
        if (a.resets && t >= 0 && a.resets[b * a.rb + t * a.rt])
#pragma unroll
            for (int i = 0; i < j; i++) win[i] = 0.0f;
        win[j] = input_at<T, W>(a, b, t, d);
    }
}

template <typename T, int W>
__global__ __launch_bounds__(kThreads) void conv_fwd_kernel(ConvArgs a) {
    const long long item = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int d = (int)(item % a.D);
    const long long row = item / a.D;                    // (b, run)
    if (row >= (long long)a.B * a.runs) return;
    const int b = (int)(row / a.runs), t0 = (int)(row % a.runs) * kRun;
    const int len = seq_len(a.lengths, b, a.T);
    const int t1 = min(t0 + kRun, a.T), tv = min(t1, len);
    T* y = (T*)a.y + ((long long)b * a.T) * a.D + d;
    float w[W], win[W];
#pragma unroll
    for (int k = 0; k < W; k++) w[k] = a.w[(long long)d * W + k];
    const float bias = a.bias ? a.bias[d] : 0.0f;
    if (t0 < tv || (len == 0 && t0 == 0)) load_window<T, W>(a, b, min(t0, len), d, win);
    for (int t = t0; t < tv; t++) {
        if (a.resets && a.resets[b * a.rb + t * a.rt])
#pragma unroll
            for (int j = 0; j < W - 1; j++) win[j] = 0.0f;
        win[W - 1] = to_f32(((const T*)a.x)[b * a.xb + t * a.xt + d]);
        float p = bias;
#pragma unroll
        for (int k = 0; k < W; k++) p = __builtin_fmaf(w[k], win[k], p);
        y[(long long)t * a.D] = from_f32<T>(a.silu ? p * sigmoid(p) : p);
#pragma unroll
        for (int j = 0; j < W - 1; j++) win[j] = win[j + 1];
    }
    for (int t = max(t0, tv); t < t1; t++) y[(long long)t * a.D] = from_f32<T>(0.0f);
    // the run that holds the last step (the first run of an empty sequence) leaves the state behind
    if (a.s1 && (len == 0 ? t0 == 0 : (t0 < len && len <= t0 + kRun))) {
        T* s1 = (T*)a.s1 + ((long long)b * (W - 1)) * a.D + d;
#pragma unroll
        for (int j = 0; j < W - 1; j++) s1[(long long)j * a.D] = from_f32<T>(win[j]);
    }
}

// dp[t] = dy[t] act'(p[t]);  dx[t] = sum_k w[k] dp[t+W-1-k], the later step not behind a reset after t.  The thread walks on W-1
// steps past its run for the contributions of later steps; those steps' own parameter gradients belong to the next run.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void conv_bwd_kernel(ConvArgs a, ConvGradArgs g) {
    const long long item = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int d = (int)(item % a.D);
    const long long lane_row = item / a.D;
    if (lane_row >= g.rows) return;
    float w[W], dw[W], db = 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) w[k] = a.w[(long long)d * W + k], dw[k] = 0.0f;
    const float bias = a.bias ? a.bias[d] : 0.0f;
    for (long long row = lane_row; row < (long long)a.B * a.runs; row += g.rows) {
        const int b = (int)(row / a.runs), t0 = (int)(row % a.runs) * kRun, t1 = min(t0 + kRun, a.T);
        const int len = seq_len(a.lengths, b, a.T);
        T* dx = (T*)g.dx + ((long long)b * a.T) * a.D + d;
        float win[W], acc[W];                      // inputs and their gradients, oldest first
#pragma unroll
        for (int j = 0; j < W; j++) acc[j] = 0.0f;
        load_window<T, W>(a, b, t0, d, win);       // beyond the length: read but not used (dp = 0 there)
        int alive = W;                             // taps that reach back over no reset since the run's start
        for (int t = t0; t < t1 + W - 1; t++) {
            float dp = 0.0f;
            win[W - 1] = 0.0f;
            if (t < len) {
                if (a.resets && a.resets[b * a.rb + t * a.rt]) {
                    alive = 1;
#pragma unroll
                    for (int j = 0; j < W - 1; j++) win[j] = 0.0f;
                }
                win[W - 1] = to_f32(((const T*)a.x)[b * a.xb + t * a.xt + d]);
                float p = bias;
#pragma unroll
                for (int k = 0; k < W; k++) p = __builtin_fmaf(w[k], win[k], p);
                dp = to_f32(((const T*)g.dy)[b * g.dyb + t * g.dyt + d]);
                if (a.silu) {
                    const float s = sigmoid(p);
                    dp *= s * (1.0f + p * (1.0f - s));
                }
                if (t < t1) {
                    db += dp;
#pragma unroll
                    for (int k = 0; k < W; k++) dw[k] = __builtin_fmaf(dp, win[k], dw[k]);
                }
#pragma unroll
                for (int k = 0; k < W; k++) acc[k] = k >= W - alive ? __builtin_fmaf(w[k], dp, acc[k]) : acc[k];
                alive = min(alive + 1, W);
            }
            const int done = t - (W - 1);          // this input has met every step that reads it
            if (g.ds1 && t >= len && done < len && len - 1 - done < alive - 1)      // ... and is part of the state left behind
                acc[0] += to_f32(((const T*)g.ds1)[((long long)b * (W - 1) + (t - len)) * a.D + d]);
            if (done >= t0) dx[(long long)done * a.D] = from_f32<T>(acc[0]);
            else if (t0 == 0 && g.ds0) ((T*)g.ds0)[((long long)b * (W - 1) + t) * a.D + d] = from_f32<T>(acc[0]);
#pragma unroll
            for (int j = 0; j < W - 1; j++) win[j] = win[j + 1], acc[j] = acc[j + 1];
            acc[W - 1] = 0.0f;
        }
    }
    float* out = g.partials + (lane_row * a.D + d) * (W + 1);
#pragma unroll
    for (int k = 0; k < W; k++) out[k] = dw[k];
    out[W] = db;
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

template <typename T, int W>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(const T* x, long long xb, T* state, const float* weight, const float* bias,
                                                            const unsigned char* resets, T* y, int B, int D, int silu) {
    const long long item = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (item >= (long long)B * D) return;
    const int b = (int)(item / D), d = (int)(item - (long long)b * D);
    T* s = state + (long long)b * (W - 1) * D + d;
    const bool cut = resets && resets[b];
    const T now = x[b * xb + d];
    T win[W];
#pragma unroll
    for (int j = 0; j < W - 1; j++) win[j] = cut ? from_f32<T>(0.0f) : s[(long long)j * D];
    win[W - 1] = now;
    float p = bias ? bias[d] : 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) p = __builtin_fmaf(weight[(long long)d * W + k], to_f32(win[k]), p);
    y[item] = from_f32<T>(silu ? p * sigmoid(p) : p);
#pragma unroll
    for (int j = 0; j < W - 1; j++) s[(long long)j * D] = win[j + 1];
}

int runs_of(int T) { return (T + kRun - 1) / kRun; }

// rows of partial parameter gradients: enough threads to fill the chip, and no more rows than there are runs
int grad_rows(long long B, int T, int D) {
    const long long all = B * runs_of(T), want = (262144 + D - 1) / D;
    return (int)(all < want ? all : want);
}

int check(const ag_conv_args* p) {
    if (!p || p->struct_size != sizeof(ag_conv_args) || !p->x_dev || !p->weight_dev) return AG_ERR_INVALID_ARG;
    if (p->B <= 0 || p->T <= 0 || p->D <= 0) return AG_ERR_INVALID_ARG;
    if (p->W < 2 || p->W > 8 || p->dtype < AG_F32 || p->dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    if (((long long)p->B * runs_of(p->T) * p->D + kThreads - 1) / kThreads > 0x7fffffffLL) return AG_ERR_UNSUPPORTED;
    return AG_OK;
}

ConvArgs device_args(const ag_conv_args* p) {
    return ConvArgs{p->x_dev, p->weight_dev, p->bias_dev, p->state_in_dev, p->lengths_dev, p->resets_dev, p->y_dev, p->state_out_dev,
                    p->x_sb, p->x_st, p->r_sb, p->r_st, p->B, p->T, p->D, p->silu, runs_of(p->T)};
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

extern "C" int ag_causal_conv_fwd(const ag_conv_args* p, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!p->y_dev) return AG_ERR_INVALID_ARG;
    const ConvArgs a = device_args(p);
    const long long items = (long long)a.B * a.runs * a.D;
    const dim3 grid((unsigned)((items + kThreads - 1) / kThreads));
    AG_FOR_DTYPE(p->dtype, AG_FOR_TAPS(p->W, hipLaunchKernelGGL((conv_fwd_kernel<T, W>), grid, dim3(kThreads), 0, (hipStream_t)stream, a)));
    return seq_status();
}

extern "C" long long ag_causal_conv_workspace_bytes(int B, int T, int D, int W) {
    if (B <= 0 || T <= 0 || D <= 0 || W < 2 || W > 8) return 0;
    return (long long)grad_rows(B, T, D) * D * (W + 1) * (long long)sizeof(float);
}

extern "C" int ag_causal_conv_bwd(const ag_conv_args* p, const ag_conv_grads* q, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!q || q->struct_size != sizeof(ag_conv_grads) || !q->dy_dev || !q->dx_dev || !q->dweight_dev || !q->workspace_dev)
        return AG_ERR_INVALID_ARG;
    if (q->workspace_bytes < ag_causal_conv_workspace_bytes(p->B, p->T, p->D, p->W)) return AG_ERR_INVALID_ARG;
    const ConvArgs a = device_args(p);
    const int rows = grad_rows(a.B, a.T, a.D);
    const ConvGradArgs g{q->dy_dev, q->dstate_out_dev, q->dx_dev, q->dstate_dev, (float*)q->workspace_dev, q->dy_sb, q->dy_st, rows};
    const dim3 grid((unsigned)(((long long)rows * a.D + kThreads - 1) / kThreads));
    AG_FOR_DTYPE(p->dtype, AG_FOR_TAPS(p->W, hipLaunchKernelGGL((conv_bwd_kernel<T, W>), grid, dim3(kThreads), 0, (hipStream_t)stream, a, g)));
    launch_sum_rows(g.partials, rows, (long long)a.D * (p->W + 1), ConvParams{q->dweight_dev, q->dbias_dev, p->W}, stream);
    return seq_status();
}

extern "C" int ag_causal_conv_step(const void* x, long long x_sb, void* state, const float* weight, const float* bias,
                                   const unsigned char* resets, void* y, int dtype, int B, int D, int W_, int silu, void* stream) {
    if (!x || !state || !weight || !y || B <= 0 || D <= 0) return AG_ERR_INVALID_ARG;
    if (W_ < 2 || W_ > 8 || dtype < AG_F32 || dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    const long long blocks = ((long long)B * D + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL) return AG_ERR_UNSUPPORTED;
    AG_FOR_DTYPE(dtype, AG_FOR_TAPS(W_, hipLaunchKernelGGL((conv_step_kernel<T, W>), dim3((unsigned)blocks), dim3(kThreads), 0,
                                                           (hipStream_t)stream, (const T*)x, x_sb, (T*)state, weight, bias, resets, (T*)y,
                                                           B, D, silu)));
    return seq_status();
}
