// policy_loss.hip - clipped policy loss with a KL term over rows of logits, and the log-probability of a row's action.
//
//   lp = x_a - lse,  lse = m + log S,  S = sum e^{x-m},  H = log S - (sum e^{x-m} (x-m)) / S
//   row loss = max(-A r, -A clip(r)) + kl (e^d - d - 1) - ent H,   r = e^{lp - old},  d = ref - lp
//   d loss / d x_j = f (delta_ja - p_j) + ent p_j (log p_j + H),   f = [-A r if the unclipped side is the larger] + kl (1 - e^d)
//
// One workgroup per row: a first sweep forms the maximum and, against it, the two sums (each thread against a maximum of its own,
// joined at the end); a second one, which finds the row in the cache, writes the gradient.  Logits of -inf have probability 0; where
// 0 times their infinite log-probability would appear, the log-probability is held at -1e30 instead.
#include "seq_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr float kFloor = -1e30f;
constexpr int kSums = 5;               // policy loss, KL term, entropy, KL of the old policy, clipped

struct LossArgs {
    const void* logits; const long long* actions; const float *old_logp, *adv, *ref_logp; const unsigned char* mask;
    void* dlogits; const float* count;
    float* rows;                       // [R, kSums] per-row terms
    float *logp, *entropy;
    long long R1, s0, s1, R;
    int V;
    float e_clip, kl_coef, entropy_coef;
};

struct Sums { float m, s, t; };        // maximum, sum e^{x-m}, sum e^{x-m} (x-m)

__device__ __forceinline__ float safe_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m), base = safe_max(m);
    const float da = fmaxf(a.m - base, kFloor), dbb = fmaxf(b.m - base, kFloor);
    const float ea = exp_hw(da), eb = exp_hw(dbb);
    // t shifts with the base: sum e^{x-m} (x-m) = e^{a.m-m} (a.t + (a.m-m) a.s)
    return Sums{m, a.s * ea + b.s * eb, ea * (a.t + da * a.s) + eb * (b.t + dbb * b.s)};
}

__device__ __forceinline__ Sums wave_join(Sums v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = join(v, Sums{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)});
    return v;
}

// a row's loss terms and the two coefficients of its gradient
struct Row { float lse, H, f, ent; };

template <typename T>
__global__ __launch_bounds__(kThreads) void token_loss_kernel(LossArgs a) {
    __shared__ Sums part[kThreads / 64];
    const long long row = blockIdx.x;
    const T* x = (const T*)a.logits + (row / a.R1) * a.s0 + (row % a.R1) * a.s1;
    T* dx = a.dlogits ? (T*)a.dlogits + row * a.V : nullptr;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (a.mask && !a.mask[row]) {
        if (dx)
            for (int j = threadIdx.x; j < a.V; j += kThreads) dx[j] = from_f32<T>(0.0f);
        if (threadIdx.x < kSums && a.rows) a.rows[row * kSums + threadIdx.x] = 0.0f;
        return;
    }
    Sums v{-__builtin_inff(), 0.0f, 0.0f};
    for (int j = threadIdx.x; j < a.V; j += kThreads) {
        const float xv = to_f32(x[j]);
        const float m = fmaxf(v.m, xv);
        if (m != v.m) v = join(v, Sums{m, 0.0f, 0.0f});
        const float e = exp_hw(xv - safe_max(v.m));
        v.s += e;
        v.t = __builtin_fmaf(e, fmaxf(xv - safe_max(v.m), kFloor), v.t);
    }
    v = wave_join(v);
    if (lane == 0) part[w] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; i++) v = join(v, part[i]);
    const float logS = log2_hw(v.s) * kLn2, base = safe_max(v.m), H = logS - v.t / v.s;
    const long long act = a.actions[row];
    const float lp = act >= 0 && act < a.V ? (to_f32(x[act]) - base) - logS : __builtin_nanf("");
    if (a.logp) {
        if (threadIdx.x == 0) {
            a.logp[row] = lp;
            if (a.entropy) a.entropy[row] = H;
        }
        return;
    }
    const float adv = a.adv[row], moved = lp - a.old_logp[row], r = expf(moved);
    const float rc = fminf(fmaxf(r, 1.0f - a.e_clip), 1.0f + a.e_clip);
    const float plain = -adv * r, held = -adv * rc;
    float kl = 0.0f, f = plain >= held || !(plain == plain) ? plain : 0.0f;
    if (a.ref_logp) {
        const float d = a.ref_logp[row] - lp, em = expm1f(d);
        kl = em - d;
        f -= a.kl_coef * em;
    }
    if (threadIdx.x == 0) {
        float* t = a.rows + row * kSums;
        t[0] = plain != plain ? plain : fmaxf(plain, held);
        t[1] = kl;
        t[2] = H;
        t[3] = expm1f(moved) - moved;
        t[4] = r < 1.0f - a.e_clip || r > 1.0f + a.e_clip ? 1.0f : 0.0f;
    }
    if (!dx) return;
    const float n = 1.0f / a.count[0], ent = a.entropy_coef * n;
    f *= n;
    for (int j = threadIdx.x; j < a.V; j += kThreads) {
        const float lj = fmaxf((to_f32(x[j]) - base) - logS, kFloor), xj = to_f32(x[j]);
        const float p = exp_hw((xj - base) - logS);
        float gj = p * (ent * (lj + H) - f);
        if (j == act) gj += f;
        if (lp != lp) gj = lp;
        dx[j] = from_f32<T>(gj);
    }
}

// number of rows that count, at least 1
__global__ __launch_bounds__(1024) void count_kernel(const unsigned char* mask, long long R, float* count) {
    __shared__ int part[16];
    int c = 0;
    for (long long i = threadIdx.x; i < R; i += 1024) c += mask ? mask[i] != 0 : 1;
    for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        for (int i = 0; i < 16; i++) s += part[i];
        count[0] = s > 0 ? (float)s : 1.0f;
        count[1] = (float)s;
    }
}

__global__ __launch_bounds__(1024) void stats_kernel(const float* rows, long long R, const float* count, float kl_coef, float ent_coef,
                                                     float* stats) {
    __shared__ double part[16][kSums];
    double s[kSums] = {0, 0, 0, 0, 0};
    for (long long i = threadIdx.x; i < R; i += 1024)
        for (int k = 0; k < kSums; k++) s[k] += rows[i * kSums + k];
    for (int k = 0; k < kSums; k++) {
        for (int o = 32; o; o >>= 1) s[k] += __shfl_xor(s[k], o);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][k] = s[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double t[kSums];
        for (int k = 0; k < kSums; k++) {
            t[k] = 0;
            for (int i = 0; i < 16; i++) t[k] += part[i][k];
            t[k] /= (double)count[0];
        }
        stats[0] = (float)(t[0] + (double)kl_coef * t[1] - (double)ent_coef * t[2]);
        for (int k = 0; k < kSums; k++) stats[1 + k] = (float)t[k];
        stats[6] = count[1];
        stats[7] = 0.0f;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(T* x, long long n, const float* scale) {
    const float g = scale[0];
    if (g == 1.0f) return;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) x[i] = from_f32<T>(to_f32(x[i]) * g);
}

}  // namespace

extern "C" long long ag_token_policy_loss_workspace_bytes(long long R, int V) {
    if (R <= 0 || V <= 0) return 0;
    return (4 + R * kSums) * (long long)sizeof(float);
}

extern "C" int ag_token_policy_loss(const ag_token_loss_args* p, void* stream) {
    if (!p || p->struct_size != sizeof(ag_token_loss_args) || !p->logits_dev || !p->actions_dev || !p->old_logp_dev || !p->advantages_dev ||
        !p->stats_dev || !p->workspace_dev || p->R0 <= 0 || p->R1 <= 0 || p->V <= 0)
        return AG_ERR_INVALID_ARG;
    if (p->dtype < AG_F32 || p->dtype > AG_F16 || p->R0 > 0x7fffffffLL / p->R1) return AG_ERR_UNSUPPORTED;
    const long long R = p->R0 * p->R1;
    if (p->workspace_bytes < ag_token_policy_loss_workspace_bytes(R, p->V)) return AG_ERR_INVALID_ARG;
    float* count = (float*)p->workspace_dev;
    const LossArgs a{p->logits_dev, p->actions_dev, p->old_logp_dev, p->advantages_dev, p->ref_logp_dev, p->mask_dev, p->dlogits_dev, count,
                     count + 4, nullptr, nullptr, p->R1, p->s0, p->s1, R, p->V, p->e_clip, p->kl_coef, p->entropy_coef};
    hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, p->mask_dev, R, count);
    AG_FOR_DTYPE(p->dtype, hipLaunchKernelGGL((token_loss_kernel<T>), dim3((unsigned)R), dim3(kThreads), 0, (hipStream_t)stream, a));
    hipLaunchKernelGGL(stats_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a.rows, R, count, p->ref_logp_dev ? p->kl_coef : 0.0f,
                       p->entropy_coef, p->stats_dev);
    return seq_status();
}

extern "C" int ag_token_logp(const void* logits, long long R0, long long R1, long long s0, long long s1, int V, int dtype,
                             const long long* actions, float* logp, float* entropy, void* stream) {
    if (!logits || !actions || !logp || R0 <= 0 || R1 <= 0 || V <= 0) return AG_ERR_INVALID_ARG;
    if (dtype < AG_F32 || dtype > AG_F16 || R0 > 0x7fffffffLL / R1) return AG_ERR_UNSUPPORTED;
    const LossArgs a{logits, actions, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, logp, entropy, R1, s0, s1, R0 * R1, V,
                     0.0f, 0.0f, 0.0f};
    AG_FOR_DTYPE(dtype, hipLaunchKernelGGL((token_loss_kernel<T>), dim3((unsigned)a.R), dim3(kThreads), 0, (hipStream_t)stream, a));
    return seq_status();
}

extern "C" int ag_scale_by(void* x, long long n, int dtype, const float* scale, void* stream) {
    if (!x || !scale || n <= 0) return AG_ERR_INVALID_ARG;
    if (dtype < AG_F32 || dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    const long long blocks = (n + 255) / 256;
    AG_FOR_DTYPE(dtype, hipLaunchKernelGGL((scale_kernel<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, (hipStream_t)stream,
                                           (T*)x, n, scale));
    return seq_status();
}
