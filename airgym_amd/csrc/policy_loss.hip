// policy_loss.hip - clipped policy loss with a KL term over rows of logits, and the log-probability of a row's action.
//
//   lp = x_a - lse,  lse = m + log S,  S = sum e^{x-m},  H = log S - (sum e^{x-m} (x-m)) / S
//   row loss = max(-A r, -A clip(r)) + kl (e^d - d - 1) - ent H,   r = e^{lp - old},  d = ref - lp
//   d loss / d x_j = f (delta_ja - p_j) + ent p_j (log p_j + H),   f = [-A r if the unclipped side is the larger] + kl (1 - e^d)
//
// Read once, write once: a row is held in registers, 16 bytes per access, between the sums and the gradient - by 1 to 64 lanes of a
// wave (short rows), by a workgroup of 256 or 1024 threads, or, beyond what registers hold, read a second time from the cache.
// Every wave sums against a maximum of its own and the waves' results are joined.  Memory bounds it in float32: 8192 x 32000 with the
// gradient takes 360 us = 5.8 TB/s, the log-probabilities alone 177 us = 5.9 TB/s.  In the 16-bit types the two exponentials and some 15
// other instructions per element bound it as much: 8192 x 32000 bfloat16 takes 218 us = 4.8 TB/s, the vector pipe busy for 81 % of it.
// float16 logits under autograd are the exception: a row's factors span more than their type does - a mean over many rows is below 6e-8 where
// a single row's ratio may be above 65504 -, so that their gradient cannot be rounded before what the loss is scaled by is known.  The
// forward leaves a copy of the logits and each row's factors, the backward forms the gradient in the copy's place, rounded once.
// Logits of -inf have probability 0.  Their infinite log-probability would meet it as 0 times inf: a wave that finds its second sum
// NaN forms it again with the log-probability held at -1e30; the gradient holds it there always.
#include "seq_common.hpp"

namespace {

constexpr float kFloor = -1e30f;
constexpr int kSums = 5;               // policy loss, KL term, entropy, KL of the old policy, clipped

// what a row's gradient is formed from later: `act` < 0 is an action out of range, kUncounted a row that does not count
struct KeptRow { float base, lS, f, k, ent; int act, pad[2]; };
static_assert(sizeof(KeptRow) == AG_TOKEN_KEPT_ROW_FLOATS * sizeof(float), "a row of kept_rows_dev");
constexpr int kUncounted = -2;

struct LossArgs {
    const void* logits; const long long* actions; const float *old_logp, *adv, *ref_logp; const unsigned char* mask;
    void* dlogits; const float* count; // {max(rows that count, 1), rows that count, 1 / the first}, or NULL: all R
    float4* rows;                      // [R] what the statistics need of a row: its action's logit, the base, the two sums
    float *logp, *entropy;             // the log-probability form: these instead
    long long R1, s0, s1, R;
    int V;
    float e_clip, kl_coef, entropy_coef, inv_R;
    KeptRow* kept;                     // [R], float16: dlogits gets the logits themselves, this what their gradient takes besides; or NULL
};

// 1 / rows that count
__device__ __forceinline__ float share_of(const LossArgs& a) { return a.count ? a.count[2] : a.inv_R; }
// whether the logits are kept for a later gradient (compiled for float16 only)
template <typename T> __device__ __forceinline__ bool keeps(const LossArgs& a) { return __is_same(T, f16_t) && a.kept; }

// x of the lane that differs in bit 0, 1 (of a lane's four), 2 (mirrored within eight), 3 (within sixteen): no LDS, one instruction
template <int kCtrl> __device__ __forceinline__ float across(float x) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), kCtrl, 0xf, 0xf, true));
}
// op over each L lanes in a row, in all of them; 64: the wave, all of whose lanes are here
template <int L, typename Op> __device__ __forceinline__ float over_lanes(float x, Op op) {
    if (L > 1) x = op(x, across<0xB1>(x));
    if (L > 2) x = op(x, across<0x4E>(x));
    if (L > 4) x = op(x, across<0x141>(x));
    if (L > 8) x = op(x, across<0x140>(x));
    if (L > 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    if (L > 32) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    return x;
}
template <int L> __device__ __forceinline__ float max_over(float x) { return over_lanes<L>(x, [](float a, float b) { return fmaxf(a, b); }); }
template <int L> __device__ __forceinline__ float sum_over(float x) { return over_lanes<L>(x, [](float a, float b) { return a + b; }); }

// e^x to about 2 ulp: 2^y, y = x log2(e) rounded, times 1 + what the rounding and log2(e)'s own left out.  A row's factors are formed by
// every lane of its waves, so that the general functions' tables of cases were most of a short row's work.
__device__ __forceinline__ float exp_near(float x) {
    const float y = x * kLog2e, r = exp2_hw(y), lost = __builtin_fmaf(x, 1.925963e-8f, __builtin_fmaf(x, kLog2e, -y));
    return __builtin_fabsf(x) < 128.0f ? r * __builtin_fmaf(lost, kLn2, 1.0f) : r;
}
// e^x - 1: below 0.35 by its series, whose next term is below 2^-26 of the sum
__device__ __forceinline__ float expm1_near(float x) {
    float p = 1.0f / 5040.0f;
    p = __builtin_fmaf(p, x, 1.0f / 720.0f);
    p = __builtin_fmaf(p, x, 1.0f / 120.0f);
    p = __builtin_fmaf(p, x, 1.0f / 24.0f);
    p = __builtin_fmaf(p, x, 1.0f / 6.0f);
    p = __builtin_fmaf(p, x, 0.5f);
    return __builtin_fabsf(x) < 0.35f ? __builtin_fmaf(p * x, x, x) : exp_near(x) - 1.0f;
}

// a x, and 0 where a is 0 and x beyond the type: an advantage or a coefficient of exactly zero takes its term out (NaN stays)
template <typename F> __device__ __forceinline__ F times(F a, F x) { return a == 0 && __builtin_isinf(x) ? (F)0 : a * x; }

struct Sums { float m, s, t; };        // with y = (x - m) log2(e), m the maximum: m, sum 2^y, sum 2^y y

// (x - m first: with y as one FMA, x log2(e) - c, the rounding of c would be all of y where every logit of a row is a mask's -1e30)
__device__ __forceinline__ float safe_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float shifted(float x, float base) { return (x - base) * kLog2e; }

__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m), base = safe_max(m);
    const float da = fmaxf(shifted(a.m, base), kFloor), db = fmaxf(shifted(b.m, base), kFloor);
    const float ea = exp2_hw(da), eb = exp2_hw(db);
    // t shifts with the base: sum 2^(y + da) (y + da) = 2^da (t + da s)
    return Sums{m, a.s * ea + b.s * eb, ea * (a.t + da * a.s) + eb * (b.t + db * b.s)};
}

template <typename T> __device__ __forceinline__ const T* row_of(const LossArgs& a, long long row) {
    const unsigned i = (unsigned)row / (unsigned)a.R1;         // R0 R1 < 2^31
    return (const T*)a.logits + i * a.s0 + (row - (long long)i * a.R1) * a.s1;
}

// what a row's sums say: base and log2 of the softmax's sum, entropy, log-probability, and the factors of its gradient
struct Row {
    float base, lS, H, lp, f, k, ent;  // p (ent log2 p + k), and f for the action
};

__device__ __forceinline__ Row finish_row(const LossArgs& a, Sums v, float xa, long long row) {
    Row r;
    r.base = safe_max(v.m);
    r.lS = log2_hw(v.s);
    r.H = (r.lS - v.t * rcp_hw(v.s)) * kLn2;
    r.lp = (xa - r.base) - r.lS * kLn2;
    r.f = r.k = r.ent = 0.0f;
    if (a.logp) return r;
    const float adv = a.adv[row], ratio = exp_near(r.lp - a.old_logp[row]);
    const float held = -adv * fminf(fmaxf(ratio, 1.0f - a.e_clip), 1.0f + a.e_clip), plain = times(-adv, ratio);
    float f = plain >= held || plain != plain ? plain : 0.0f;
    if (a.ref_logp && a.kl_coef != 0.0f) f -= a.kl_coef * expm1_near(a.ref_logp[row] - r.lp);
    const float n = share_of(a);
    r.f = f * n;
    r.ent = a.entropy_coef * n * kLn2;
    r.k = __builtin_fmaf(a.entropy_coef * n, r.H, -r.f);
    return r;
}

// f (delta - p) + ent p (log p + H) without the delta
template <typename R> __device__ __forceinline__ float grad_of(const R& r, float x) {
    const float q = fmaxf(__builtin_fmaf(x - r.base, kLog2e, -r.lS), kFloor);      // log2 p
    return exp2_hw(q) * __builtin_fmaf(r.ent, q, r.k);
}

// one element's share of the sums
__device__ __forceinline__ void add_to(Sums& v, float x, float base) {
    const float y = shifted(x, base), e = exp2_hw(y);
    v.s += e;
    v.t = __builtin_fmaf(e, y, v.t);
}

// ---- short rows: L lanes of a wave per row, up to 8 elements a lane ------------------------------------------------------
constexpr int kShortThreads = 256, kPerLane = 8, kShortLanes = 32;

template <typename T, int L>
__global__ __launch_bounds__(kShortThreads) void token_loss_short_kernel(LossArgs a) {
    constexpr int kRows = kShortThreads / L;
    const int l = threadIdx.x % L;
    const long long row = (long long)blockIdx.x * kRows + threadIdx.x / L;
    const bool there = row < a.R, on = there && !(a.mask && !a.mask[row]);
    float x[kPerLane], xa = __builtin_nanf("");
    Row r;
    int act = -1;
    if (on) {
        const T* p = row_of<T>(a, row);
        const long long av = a.actions[row];
        act = av >= 0 && av < a.V ? (int)av : -1;
        float m = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < kPerLane; k++) {
            const int j = l + k * L;
            x[k] = j < a.V ? to_f32(p[j]) : -__builtin_inff();
            m = fmaxf(m, x[k]);
        }
        if (act >= 0) xa = to_f32(p[act]);
        m = max_over<L>(m);
        Sums v{m, 0.0f, 0.0f};
        const float base = safe_max(m);
#pragma unroll
        for (int k = 0; k < kPerLane; k++)
            if (l + k * L < a.V) {
                const float y = shifted(x[k], base), e = exp2_hw(y);
                v.s += e;
                v.t = __builtin_fmaf(e, fmaxf(y, kFloor), v.t);
            }
        v.s = sum_over<L>(v.s), v.t = sum_over<L>(v.t);
        r = finish_row(a, v, xa, row);
        if (!a.logp && l == 0) a.rows[row] = float4{xa, r.base, v.s, v.t};
        if (a.logp) {
            if (l == 0) {
                a.logp[row] = r.lp;
                if (a.entropy) a.entropy[row] = r.H;
            }
        }
    }
    if (keeps<T>(a) && there && l == 0) a.kept[row] = on ? KeptRow{r.base, r.lS, r.f, r.k, r.ent, act, {0, 0}} : KeptRow{0, 0, 0, 0, 0, kUncounted, {0, 0}};
    if (a.dlogits && there) {
        T* dx = (T*)a.dlogits + row * a.V;
#pragma unroll
        for (int k = 0; k < kPerLane; k++) {
            const int j = l + k * L;
            if (j < a.V) {
                float g = 0.0f;
                if (on) g = keeps<T>(a) ? x[k] : grad_of(r, x[k]) + (j == act ? r.f : 0.0f);
                dx[j] = from_f32<T>(g);
            }
        }
    }
}

// ---- long rows: a workgroup per row -----------------------------------------------------------------------------------------
// NV > 0: the row is held in NV accesses per thread.  NV = 0: it is longer than that, and read again for the gradient.
// kOnceIn, kOnceOut: logits, gradients that the caches will not keep.
template <typename T, int THREADS, int NV, bool kOnceIn, bool kOnceOut>
__global__ __launch_bounds__(THREADS) void token_loss_kernel(LossArgs a) {
    constexpr int E = 16 / sizeof(T), kWaves = THREADS / 64, kKeep = NV ? NV : 1;
    __shared__ Sums part[kWaves];
    const long long row = blockIdx.x;
    const T* x = row_of<T>(a, row);
    T* dx = a.dlogits ? (T*)a.dlogits + row * a.V : nullptr;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int full = a.V / E, nq = NV ? NV : (full + THREADS - 1) / THREADS;      // whole accesses of the row, per thread
    const int tail = full * E + threadIdx.x;                                        // the elements behind them: one per thread
    if (a.mask && !a.mask[row]) {
        if (keeps<T>(a)) {
            if (threadIdx.x == 0) a.kept[row] = KeptRow{0, 0, 0, 0, 0, kUncounted, {0, 0}};
            return;
        }
        const Vec<T, E> zero{{0, 0, 0, 0}};
        if (dx) {
            for (int q = threadIdx.x; q < full; q += THREADS) store_vec<T, E, kOnceOut>(dx + q * E, zero);
            if (tail < a.V) dx[tail] = from_f32<T>(0.0f);
        }
        return;
    }
    const long long av = a.actions[row];
    const int act = av >= 0 && av < a.V ? (int)av : -1;
    const float xa = act >= 0 ? to_f32(x[act]) : __builtin_nanf("");
    Vec<T, E> c[kKeep];
    Sums v{-__builtin_inff(), 0.0f, 0.0f};
    // The row stays as it came: without this the compiler keeps the 16-bit types' float forms from one pass over it to the next, two
    // registers for one.
    auto as_it_came = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kKeep; k++) asm volatile("" : "+v"(c[k].w[0]), "+v"(c[k].w[1]), "+v"(c[k].w[2]), "+v"(c[k].w[3]));
    };
    // the sums of what c (and xt) holds against the wave's maximum m, joined to what the wave has
    auto sum_up = [&](int k0, float xt) __attribute__((always_inline)) {
        float m = xt;
#pragma unroll
        for (int k = 0; k < kKeep; k++)
            if ((k0 + k) * THREADS + (int)threadIdx.x < full)
#pragma unroll
                for (int i = 0; i < E; i++) m = fmaxf(m, c[k].at(i));
        m = max_over<64>(m);
        Sums u{m, 0.0f, 0.0f};
        const float base = safe_max(m);
        as_it_came();
#pragma unroll
        for (int k = 0; k < kKeep; k++)
            if ((k0 + k) * THREADS + (int)threadIdx.x < full)
#pragma unroll
                for (int i = 0; i < E; i++) add_to(u, c[k].at(i), base);
        if (u.t != u.t) {              // some y are -inf (or NaN, which stays)
            u.t = 0.0f;
            as_it_came();
#pragma unroll
            for (int k = 0; k < kKeep; k++)
                if ((k0 + k) * THREADS + (int)threadIdx.x < full)
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        const float y = shifted(c[k].at(i), base);
                        u.t = __builtin_fmaf(exp2_hw(y), fmaxf(y, kFloor), u.t);
                    }
        }
        if (k0 == 0 && tail < a.V) {
            const float y = shifted(xt, base), e = exp2_hw(y);
            u.s += e;
            u.t = __builtin_fmaf(e, fmaxf(y, kFloor), u.t);
        }
        u.s = sum_over<64>(u.s), u.t = sum_over<64>(u.t);
        v = NV ? u : join(v, u);
    };
    const float xt = tail < a.V ? to_f32(x[tail]) : -__builtin_inff();
    if constexpr (NV > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; k++) {
            const int q = threadIdx.x + k * THREADS;
            if (q < full) c[k] = load_vec<T, E, kOnceIn>(x + q * E);
        }
        sum_up(0, xt);
    } else {
        for (int k = 0; k < nq; k++) {
            const int q = threadIdx.x + k * THREADS;
            if (q < full) c[0] = load_vec<T, E>(x + q * E);
            sum_up(k, k ? -__builtin_inff() : xt);
        }
    }
    if (lane == 0) part[w] = v;
    __syncthreads();
    v = part[lane % kWaves];
#pragma unroll
    for (int o = kWaves / 2; o; o >>= 1) v = join(v, Sums{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)});
    const Row r = finish_row(a, v, xa, row);
    if (a.logp) {
        if (threadIdx.x == 0) {
            a.logp[row] = r.lp;
            if (a.entropy) a.entropy[row] = r.H;
        }
        return;
    }
    if (threadIdx.x == 0) {
        a.rows[row] = float4{xa, r.base, v.s, v.t};
        if (keeps<T>(a)) a.kept[row] = KeptRow{r.base, r.lS, r.f, r.k, r.ent, act, {0, 0}};
    }
    if (!dx) return;
    const int aq = act >= 0 ? act / E : -1, ai = act % E;
    auto gradient = [&](int q, const Vec<T, E>& held) __attribute__((always_inline)) {
        if (q >= full) return;
        if (keeps<T>(a)) {
            store_vec<T, E, kOnceOut>(dx + q * E, held);
            return;
        }
        float g[E];
#pragma unroll
        for (int i = 0; i < E; i++) g[i] = grad_of(r, held.at(i));
        if (q == aq)
#pragma unroll
            for (int i = 0; i < E; i++) g[i] += i == ai ? r.f : 0.0f;
        Vec<T, E> out;
        out.set(g);
        store_vec<T, E, kOnceOut>(dx + q * E, out);
    };
    if constexpr (NV > 0) {
        as_it_came();
#pragma unroll
        for (int k = 0; k < kKeep; k++) gradient(threadIdx.x + k * THREADS, c[k]);
    } else {
        for (int q = threadIdx.x; q < full; q += THREADS) gradient(q, load_vec<T, E>(x + q * E));
    }
    if (tail < a.V) dx[tail] = from_f32<T>(keeps<T>(a) ? xt : grad_of(r, xt) + (tail == act ? r.f : 0.0f));
}

__global__ __launch_bounds__(1024) void count_kernel(const unsigned char* mask, long long R, float* count) {
    __shared__ int part[16];
    int c = 0;
    const long long head = (16 - ((uintptr_t)mask & 15)) & 15, n16 = R > head ? (R - head) / 16 : 0;
    const uint4* m = (const uint4*)(mask + head);
    for (long long i = threadIdx.x; i < n16; i += 1024) {
        const uint4 v = m[i];
        const unsigned q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) c += __popc((q[k] | ((q[k] & 0x7f7f7f7fu) + 0x7f7f7f7fu)) & 0x80808080u);      // bytes that are not zero
    }
    if (threadIdx.x < head && threadIdx.x < R) c += mask[threadIdx.x] != 0;
    const long long tail = head + n16 * 16 + threadIdx.x;      // at most 15 bytes
    if (tail < R) c += mask[tail] != 0;
    for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        for (int i = 0; i < 16; i++) s += part[i];
        count[0] = s > 0 ? (float)s : 1.0f;
        count[1] = (float)s;
        count[2] = 1.0f / count[0];
    }
}

// The loss and its statistics: the rows' terms formed and summed in double, in an order that R alone fixes.  The terms cancel - the
// advantages have both signs -, so that float32's last bits of a log-probability of -10 would be the loss's fifth digit.  A row per
// thread: three double functions a row are work for all lanes here, and would stall a workgroup per row up there.
constexpr int kStatsThreads = 256, kStatsBlocks = 1024, kOneStage = 512, kOneStageRows = 1024;

// e^x - 1 - x from e^x - 1, infinite at both ends
__device__ __forceinline__ double beyond(double em1, double x) { return em1 == __builtin_inf() ? em1 : em1 - x; }

__device__ __forceinline__ void add_row(const LossArgs& a, long long row, double* s) {
    if (a.mask && !a.mask[row]) return;
    const float4 v = a.rows[row];
    // The sums are those of the softmax of x (1 + tilt), log2(e) being a float: log S is off by tilt times the mean x - base.
    constexpr double ln2 = 0.6931471805599453094, tilt = (double)kLog2e * ln2 - 1.0;
    const double mean = (double)v.w / v.z * ln2, logS = log((double)v.z) - tilt * mean;
    const double lp = ((double)v.x - v.y) - logS, adv = a.adv[row], moved = lp - a.old_logp[row], up = expm1(moved);
    const double ratio = 1.0 + up, low = 1.0 - (double)a.e_clip, high = 1.0 + (double)a.e_clip;
    const double held = -adv * fmin(fmax(ratio, low), high), plain = times(-adv, ratio);
    s[0] += plain != plain ? plain : fmax(plain, held);
    if (a.ref_logp) {
        const double d = a.ref_logp[row] - lp;
        s[1] += beyond(expm1(d), d);
    }
    s[2] += logS - mean;
    s[3] += beyond(up, moved);
    s[4] += ratio < low || ratio > high ? 1.0 : 0.0;
}

template <int THREADS>
__device__ __forceinline__ void sum_block(double* s) {
    __shared__ double part[THREADS / 64][kSums];
#pragma unroll
    for (int k = 0; k < kSums; k++) {
        for (int o = 32; o; o >>= 1) s[k] += __shfl_xor(s[k], o);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][k] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSums; k++) {
        s[k] = part[0][k];
#pragma unroll
        for (int i = 1; i < THREADS / 64; i++) s[k] += part[i][k];
    }
}

__global__ __launch_bounds__(kStatsThreads) void stats_part_kernel(LossArgs a, double* out) {
    double s[kSums] = {0, 0, 0, 0, 0};
    for (long long i = (long long)blockIdx.x * kStatsThreads + threadIdx.x; i < a.R; i += (long long)gridDim.x * kStatsThreads) add_row(a, i, s);
    sum_block<kStatsThreads>(s);
    if (threadIdx.x == 0)
#pragma unroll
        for (int k = 0; k < kSums; k++) out[blockIdx.x * kSums + k] = s[k];
}

// parts: the first stage's sums of `blocks` workgroups; NULL (few rows): the rows themselves
__global__ __launch_bounds__(kOneStage) void stats_kernel(LossArgs a, const double* parts, int blocks, float* loss, float* stats) {
    double s[kSums] = {0, 0, 0, 0, 0};
    if (parts) {
        for (int i = threadIdx.x; i < blocks; i += kOneStage)
#pragma unroll
            for (int k = 0; k < kSums; k++) s[k] += parts[i * kSums + k];
    } else
        for (long long i = threadIdx.x; i < a.R; i += kOneStage) add_row(a, i, s);
    sum_block<kOneStage>(s);
    if (threadIdx.x == 0) {
#pragma unroll
        for (int k = 0; k < kSums; k++) s[k] /= a.count ? (double)a.count[0] : (double)a.R, stats[k] = (float)s[k];
        loss[0] = (float)(s[0] + times((double)a.kl_coef, s[1]) - (double)a.entropy_coef * s[2]);
        stats[kSums] = a.count ? a.count[1] : (float)a.R;
    }
}

// The gradient of a loss that is not the graph's root: in bfloat16 a second rounding, unless the factor is a power of two.  (float16 has
// the kernel below.)
template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(T* x, long long n, const float* scale) {
    constexpr int E = 16 / sizeof(T);
    const float g = scale[0];
    if (g == 1.0f) return;
    const long long full = n / E, step = (long long)gridDim.x * 256, i0 = (long long)blockIdx.x * 256 + threadIdx.x;
    for (long long i = i0; i < full; i += step) {
        auto c = load_vec<T, E>(x + i * E);
        float v[E];
#pragma unroll
        for (int k = 0; k < E; k++) v[k] = c.at(k) * g;
        c.set(v);
        store_vec<T, E>(x + i * E, c);
    }
    if (full * E + i0 < n) x[full * E + i0] = from_f32<T>(to_f32(x[full * E + i0]) * g);
}

// The gradient of kept logits, in their place, times the loss's factor: rounded once.  A thread takes 16 bytes at a time wherever the rows'
// borders lie, and moves on by a fixed number of rows and columns, so that it divides once.  Its bytes bound it: 8191 x 32000 takes 195 us = 5.4 TB/s.
__global__ __launch_bounds__(256) void kept_grad_kernel(f16_t* x, const KeptRow* rows, long long n, int V, const float* scale) {
    constexpr int E = 16 / sizeof(f16_t);
    const float g = scale[0];
    const long long step = (long long)gridDim.x * 256 * E, rows_on = step / V;
    const int cols_on = (int)(step - rows_on * V);
    long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * E, row = i / V;
    int col = (int)(i - row * V);
    for (; i < n; i += step, row += rows_on, col += cols_on) {         // (col + cols_on < 2^31: V is at most 2^30)
        if (col >= V) col -= V, row++;
        const int m = n - i < E ? (int)(n - i) : E;
        Vec<f16_t, E> c;
        if (m == E) c = load_vec<f16_t, E>(x + i);
        float v[E];
        long long at = row;
        int j = col;
        KeptRow r = rows[at];
#pragma unroll
        for (int k = 0; k < E; k++) {
            if (k >= m) break;
            if (j == V) j = 0, r = rows[++at];                          // k < m: the row is there
            const float e = m == E ? c.at(k) : to_f32(x[i + k]);
            v[k] = r.act == kUncounted ? 0.0f : (grad_of(r, e) + (j == r.act ? r.f : 0.0f)) * g;
            j++;
        }
        if (m == E) {
            c.set(v);
            store_vec<f16_t, E>(x + i, c);
        } else
            for (int k = 0; k < m; k++) x[i + k] = from_f32<f16_t>(v[k]);
    }
}

}  // namespace

// Which form takes a row of V logits.  Up to 256 of them, 1 to 32 lanes share a wave with other rows (65536 x 129 float32: 26 us with the
// gradient where a wave per row takes 37; at 256 34 and 38, at 512 a wave per row moves 4.5 TB/s); beyond, a workgroup holds the row
// in accesses of 16 bytes: one wave up to 8 KB, 256 threads up to 32 KB, 1024 threads up to 256 KB; what is longer is read twice.
static int short_lanes(int V) {
    int l = 1;
    while (l <= kShortLanes && l * kPerLane < V) l *= 2;
    return l;
}

// accesses of a row
static long long accesses(int V, int size) { return ((long long)V * size + 15) / 16; }

// V up to 2^30 (element indexes run a workgroup past the row's end) and all rows in one launch
static bool launchable(long long R0, long long R1, int V, int dtype) {
    if (V > 1 << 30 || R0 > 0x7fffffffLL / R1) return false;
    const int lanes = short_lanes(V);
    const long long q = accesses(V, dtype == AG_F32 ? 4 : 2), threads = lanes <= kShortLanes ? lanes : q <= 512 ? 64 : q <= 2048 ? 256 : 1024;
    return R0 * R1 <= kMaxThreads / threads - kShortThreads;
}

template <typename T, bool IN, bool OUT>
static void launch_long_rows(const LossArgs& a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)a.R);
    const long long q = accesses(a.V, sizeof(T));
    if (q <= 64) hipLaunchKernelGGL((token_loss_kernel<T, 64, 1, IN, OUT>), grid, dim3(64), 0, st, a);
    else if (q <= 128) hipLaunchKernelGGL((token_loss_kernel<T, 64, 2, IN, OUT>), grid, dim3(64), 0, st, a);
    else if (q <= 256) hipLaunchKernelGGL((token_loss_kernel<T, 64, 4, IN, OUT>), grid, dim3(64), 0, st, a);
    else if (q <= 512) hipLaunchKernelGGL((token_loss_kernel<T, 64, 8, IN, OUT>), grid, dim3(64), 0, st, a);
    else if (q <= 1024) hipLaunchKernelGGL((token_loss_kernel<T, 256, 4, IN, OUT>), grid, dim3(256), 0, st, a);
    else if (q <= 2048) hipLaunchKernelGGL((token_loss_kernel<T, 256, 8, IN, OUT>), grid, dim3(256), 0, st, a);
    else if (q <= 4096) hipLaunchKernelGGL((token_loss_kernel<T, 1024, 4, IN, OUT>), grid, dim3(1024), 0, st, a);
    else if (q <= 8192) hipLaunchKernelGGL((token_loss_kernel<T, 1024, 8, IN, OUT>), grid, dim3(1024), 0, st, a);
    else if (q <= 16384) hipLaunchKernelGGL((token_loss_kernel<T, 1024, 16, IN, OUT>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((token_loss_kernel<T, 1024, 0, false, OUT>), grid, dim3(1024), 0, st, a);
}

template <typename T>
static void launch_rows(const LossArgs& a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const int lanes = short_lanes(a.V);
    if (lanes <= kShortLanes) {
        const int rows = kShortThreads / lanes;
        const dim3 grid((unsigned)((a.R + rows - 1) / rows)), block(kShortThreads);
        switch (lanes) {
            case 1: hipLaunchKernelGGL((token_loss_short_kernel<T, 1>), grid, block, 0, st, a); break;
            case 2: hipLaunchKernelGGL((token_loss_short_kernel<T, 2>), grid, block, 0, st, a); break;
            case 4: hipLaunchKernelGGL((token_loss_short_kernel<T, 4>), grid, block, 0, st, a); break;
            case 8: hipLaunchKernelGGL((token_loss_short_kernel<T, 8>), grid, block, 0, st, a); break;
            case 16: hipLaunchKernelGGL((token_loss_short_kernel<T, 16>), grid, block, 0, st, a); break;
            default: hipLaunchKernelGGL((token_loss_short_kernel<T, 32>), grid, block, 0, st, a); break;
        }
        return;
    }
    // The logits' writer, the loss and a reader of the gradient: 524 MB (8191 x 32000 bfloat16) 594 us plain, 594 with the logits marked as
    // used once, 552 with the gradient too; 206 MB (1023 x 50257 float32) 226, 218 and 224 us; 34 MB (1024 x 8192 float32) 47.4, 48.3 and
    // 47.5 us, without the writer 36.5, 42.5 and 42.1.
    const long long bytes = a.R * a.V * (long long)sizeof(T);
    if (bytes >= 2 * kCached) launch_long_rows<T, true, true>(a, stream);
    else if (bytes >= kCached) launch_long_rows<T, true, false>(a, stream);
    else launch_long_rows<T, false, false>(a, stream);
}

// workgroups of the statistics' first stage; 0: one stage
static int stats_blocks(long long R) {
    const long long blocks = (R + kStatsThreads - 1) / kStatsThreads;
    return R <= kOneStageRows ? 0 : (int)(blocks < kStatsBlocks ? blocks : kStatsBlocks);
}

extern "C" long long ag_token_policy_loss_workspace_bytes(long long R, int V) {
    if (R <= 0 || V <= 0) return 0;
    return 16 + R * (long long)sizeof(float4) + stats_blocks(R) * kSums * (long long)sizeof(double);
}

extern "C" int ag_token_policy_loss(const ag_token_loss_args* p, void* stream) {
    if (!p || p->struct_size != sizeof(ag_token_loss_args) || !p->logits_dev || !p->actions_dev || !p->old_logp_dev || !p->advantages_dev ||
        !p->loss_dev || !p->stats_dev || !p->workspace_dev || p->R0 <= 0 || p->R1 <= 0 || p->V <= 0)
        return AG_ERR_INVALID_ARG;
    if (p->dtype < AG_F32 || p->dtype > AG_F16 || !launchable(p->R0, p->R1, p->V, p->dtype)) return AG_ERR_UNSUPPORTED;
    if (p->kept_rows_dev && (p->dtype != AG_F16 || !p->dlogits_dev)) return AG_ERR_INVALID_ARG;
    const long long R = p->R0 * p->R1;
    if (p->workspace_bytes < ag_token_policy_loss_workspace_bytes(R, p->V)) return AG_ERR_INVALID_ARG;
    float* count = (float*)p->workspace_dev;                 // 4 floats, then the rows' sums, then the first stage's
    float4* rows = (float4*)(count + 4);
    const int blocks = stats_blocks(R);
    double* parts = blocks ? (double*)(rows + R) : nullptr;
    const LossArgs a{p->logits_dev, p->actions_dev, p->old_logp_dev, p->advantages_dev, p->ref_logp_dev, p->mask_dev, p->dlogits_dev,
                     p->mask_dev ? count : nullptr, rows, nullptr, nullptr, p->R1, p->s0, p->s1, R, p->V, p->e_clip, p->kl_coef,
                     p->entropy_coef, 1.0f / (float)R, (KeptRow*)p->kept_rows_dev};
    if (a.count) hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, p->mask_dev, R, count);
    AG_FOR_DTYPE(p->dtype, launch_rows<T>(a, stream));
    if (blocks) hipLaunchKernelGGL(stats_part_kernel, dim3((unsigned)blocks), dim3(kStatsThreads), 0, (hipStream_t)stream, a, parts);
    hipLaunchKernelGGL(stats_kernel, dim3(1), dim3(kOneStage), 0, (hipStream_t)stream, a, parts, blocks, p->loss_dev, p->stats_dev);
    return seq_status();
}

extern "C" int ag_token_logp(const void* logits, long long R0, long long R1, long long s0, long long s1, int V, int dtype,
                             const long long* actions, float* logp, float* entropy, void* stream) {
    if (!logits || !actions || !logp || R0 <= 0 || R1 <= 0 || V <= 0) return AG_ERR_INVALID_ARG;
    if (dtype < AG_F32 || dtype > AG_F16 || !launchable(R0, R1, V, dtype)) return AG_ERR_UNSUPPORTED;
    const LossArgs a{logits, actions, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, logp, entropy, R1, s0, s1, R0 * R1, V,
                     0.0f, 0.0f, 0.0f, 0.0f, nullptr};
    AG_FOR_DTYPE(dtype, launch_rows<T>(a, stream));
    return seq_status();
}

extern "C" int ag_scale_by(void* x, long long n, int dtype, const float* scale, void* stream) {
    if (!x || !scale || n <= 0) return AG_ERR_INVALID_ARG;
    if (dtype < AG_F32 || dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    const long long blocks = (n / 4 + 255) / 256 + 1;
    AG_FOR_DTYPE(dtype, hipLaunchKernelGGL((scale_kernel<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, (hipStream_t)stream,
                                           (T*)x, n, scale));
    return seq_status();
}

extern "C" int ag_token_policy_grad(void* x, const float* kept_rows, long long R, int V, int dtype, const float* scale, void* stream) {
    if (!x || !kept_rows || !scale || R <= 0 || V <= 0) return AG_ERR_INVALID_ARG;
    if (dtype != AG_F16 || !launchable(1, R, V, dtype)) return AG_ERR_UNSUPPORTED;
    const long long n = R * V, blocks = (n / 8 + 255) / 256 + 1;
    hipLaunchKernelGGL(kept_grad_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, (hipStream_t)stream, (f16_t*)x,
                       (const KeptRow*)kept_rows, n, V, scale);
    return seq_status();
}
