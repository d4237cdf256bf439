// selective_scan.hip - selective state space scan: forward, backward, single step.
//
//   dt = softplus(delta + bias);  h_t = exp(dt A) h_{t-1} + dt B_t u_t;  y_t = C_t . h_t + D u_t;  out = y z sigmoid(z)
//   (per channel d a state of N numbers; B_t, C_t shared by the channels of a group; h := 0 before a step flagged as a reset)
//
// Layout.  A workgroup owns 64 consecutive channels of one group and walks along time in tiles; wave w owns S states of all 64 channels
// (lane = channel): four waves of 1, 2 or 4 states up to N = 16, eight waves of 4 beyond.  What does not depend on the state index -
// softplus, the products dt u, the gate - is formed once per (step, channel) by whichever wave stages that row and goes through LDS; per
// (step, channel, state) there remain one multiply, one v_exp_f32, one multiply and two FMAs.  The sums over states (y, and in the
// backward the two sums behind du and ddelta) are joined through LDS, in a fixed order.
// Few rows.  When sequences and channels alone do not fill the chip, time is cut into chunks: a first pass finds what each chunk makes
// of a zero state (backward: of a zero gradient) and the sum of its time steps - exp(A sum dt) is the chunk's decay -, the main pass
// starts each chunk from those of the chunks before (behind) it.
// The vector pipe bounds the sequence kernels: v_exp_f32 takes four issue slots, so that a state costs eight per step forward and about 21
// backward (the two sums over channels among them).  At 4096 x 24 x 256, N = 16, float32, gated, with resets the forward takes 149 us
// (pipe 88 % busy; the states' slots alone are 94 us at the 2.1 GHz it runs at, its bytes 107), the backward 430 us (79 % busy; 250 us
// and 176).
#include "seq_common.hpp"

namespace {

constexpr int kTile = 16;              // steps per tile of the forward
constexpr int kBack = 8;               // steps per tile of the backward, which keeps their states in registers
constexpr int kLanes = 64;             // channels per workgroup

struct ScanArgs {
    const void *u, *delta, *z, *Bm, *Cm;
    const float *A, *Dskip, *bias, *s0;
    const int* lengths;
    const unsigned char* resets;
    long long ub, ut, db, dt, zb, zt, bb, bt, bg, cb, ct, cg, rb, rt;
    void* out;
    float *s1, *ckpt;
    float *chunk_h, *chunk_dt;         // [B, chunks, D, N], [B, chunks, D]: what a chunk makes of nothing, and its sum of dt (NaN: reset)
    int B, T, D, N, G, softplus;
    int Dg, nb;                        // channels per group, workgroups per group
    int rows;                          // forward: workgroups along the batch
    int chunks;                        // chunks of time
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

// Which 64 channels, row of the batch and chunk a workgroup has.
struct Place {
    int lane, w, g, cb, row, chunk, d0, d;      // d0: first channel of the workgroup, d: the lane's (clamped when it has none)
    bool live;
};
__device__ __forceinline__ Place place_of(const ScanArgs& a) {
    Place p;
    p.lane = threadIdx.x & 63;
    p.w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned i = blockIdx.x;
    p.cb = i % a.nb, i /= a.nb;
    p.g = i % a.G, i /= a.G;
    // With chunks a workgroup has one sequence, and all of the forward's are resident at once: a CU's, which are 256 / (nb G) apart, should
    // be of different sequences, long and short ones.
    p.chunk = a.chunks > 1 ? i / a.B : 0;
    p.row = a.chunks > 1 ? (i + p.chunk) % a.B : i;
    const int ch = p.cb * kLanes + p.lane;
    p.live = ch < a.Dg;
    p.d0 = p.g * a.Dg + p.cb * kLanes;
    p.d = p.live ? p.d0 + p.lane : p.g * a.Dg + a.Dg - 1;
    return p;
}

// The steps of a chunk: an even share, in whole tiles, of what the sequence has - shares of the padded length would leave the chunks behind
// a sequence's end idle (8 x 2047 x 2048 bf16 with lengths between 0 and T: 746 us forward and backward on average over eight draws, this
// way 666).  Without chunks: all steps, padding included.
struct Range { int from, to; };
__device__ __forceinline__ Range chunk_of(const ScanArgs& a, const Place& p) {
    if (a.chunks == 1) return Range{0, a.T};
    const int len = seq_len(a.lengths, p.row, a.T), share = ((len + a.chunks - 1) / a.chunks + kTile - 1) / kTile * kTile;
    const int from = __builtin_amdgcn_readfirstlane(p.chunk * share);
    return Range{from, __builtin_amdgcn_readfirstlane(min(from + share, len))};
}
// ... and its share of the padding from step `first` on, whose results are zero
template <typename A> __device__ __forceinline__ Range padding_of(A a, const Place& p, int first) {
    const int share = (max(a->T - first, 0) + a->chunks - 1) / a->chunks, from = first + p.chunk * share;
    return Range{from, min(from + share, a->T)};
}

// reset flags of nv steps from t0, one per lane (requested with the tile's other inputs, used a tile later)
template <typename A>
__device__ __forceinline__ unsigned char reset_flag(A a, int b, int t0, int nv, int lane) {
    return lane < nv ? a->resets[b * a->rb + (t0 + lane) * a->rt] : 0;
}
// ... and as a wave-uniform bit mask
__device__ __forceinline__ unsigned reset_bits(unsigned char flag) { return __builtin_amdgcn_readfirstlane((unsigned)__ballot(flag != 0)); }

// Resets are rare.  In the forward a reset is a branch that stays one: a select in its place would cost every step what only a reset
// needs.  The backward's tiles are written out twice, with and without them: a branch per step would keep every step's reads from LDS
// behind the step before (first pass 111 -> 100 us, main pass 390 -> 377 us at 8 x 2047 x 2048 bf16, the two at 4096 x 24 x 256 f32 with a
// reset in every 24 steps 443 -> 426 us; the forward, with 80 registers, only spills).
#define AG_RARE(cond) if (__builtin_expect(cond, 0)) if (([]() __attribute__((always_inline)) { asm volatile(""); }(), true))
template <bool B> struct Flag { static constexpr bool value = B; };
// x, or zeros (whatever x is); keep is wave-uniform
template <int S> __device__ __forceinline__ void keep_if(bool keep, float* x) {
    const unsigned mask = keep ? ~0u : 0u;
#pragma unroll
    for (int j = 0; j < S; j++) x[j] = __uint_as_float(__float_as_uint(x[j]) & mask);
}

// Addresses.  A row's base is wave-uniform and moves on by scalar adds; a lane adds 32 bits of its own (the host has checked that a
// tile of rows stays below 4 GB).  The argument block is read again, by scalar loads, where a sequence starts: all of its pointers and
// strides held at once do not fit the scalar registers, and what is spilled from them costs vector instructions.
template <typename S> using Const = const __attribute__((address_space(4))) S*;
__device__ __forceinline__ Const<ScanArgs> scan_args() {
    auto p = (Const<ScanArgs>)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
__device__ __forceinline__ Const<ScanGradArgs> grad_args() {           // the second argument, behind the first
    static_assert(sizeof(ScanArgs) % 8 == 0, "the argument blocks follow each other");
    auto p = (Const<char>)__builtin_amdgcn_kernarg_segment_ptr() + sizeof(ScanArgs);
    asm volatile("" : "+s"(p));
    return (Const<ScanGradArgs>)p;
}
struct Rows {                          // rows of a [T, ...] array from some step on
    const char* base;
    unsigned step;                     // bytes from one row to the next
    __device__ __forceinline__ void set(const void* p, long long at, long long stride, int size) {
        base = (const char*)p + at * size;
        step = (unsigned)(stride * size);
    }
    __device__ __forceinline__ void move(int rows) { base += (long long)rows * (long long)step; }
};
template <typename T> __device__ __forceinline__ T get(const Rows& x, int r, unsigned lane_bytes) {
    return *(const T*)(x.base + (r * x.step + lane_bytes));
}
template <typename T> __device__ __forceinline__ void put(char* base, unsigned bytes, T v) { *(T*)(base + bytes) = v; }

// a lane's S states (the w-th S of a row of N), zero where there are none: one access where the row is whole
typedef float two_any4 __attribute__((ext_vector_type(2), aligned(4)));
typedef float four_any4 __attribute__((ext_vector_type(4), aligned(4)));
// x[j] = c[j + by], zero beyond
__device__ __forceinline__ void shift_down(const float* c, int by, float* x) {
    x[0] = by == 0 ? c[0] : by == 1 ? c[1] : by == 2 ? c[2] : by == 3 ? c[3] : 0.0f;
    x[1] = by == 0 ? c[1] : by == 1 ? c[2] : by == 2 ? c[3] : 0.0f;
    x[2] = by == 0 ? c[2] : by == 1 ? c[3] : 0.0f;
    x[3] = by == 0 ? c[3] : 0.0f;
}
template <int S, bool kOnce = false, bool kTail = false> __device__ __forceinline__ void load_states(const float* row, int w, int N, float* x) {
    if (S == 4 && N % 4 == 0 && 4 * w < N) {
        const four_any4* at = (const four_any4*)(row + 4 * w);
        const four_any4 v = kOnce ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
        for (int j = 0; j < S; j++) x[j] = v[j];
    } else if (kTail) {                                                 // N > 4: the last lane of the row takes its last four, and what it needs of them
        const int first = min(4 * w, N - 4);
        const four_any4* at = (const four_any4*)(row + first);
        const four_any4 v = kOnce ? __builtin_nontemporal_load(at) : *at;
        const float c[4] = {v[0], v[1], v[2], v[3]};
        shift_down(c, 4 * w - first, x);
    } else if (S == 2 && N % 2 == 0 && 2 * w < N) {
        const two_any4 v = *(const two_any4*)(row + 2 * w);
#pragma unroll
        for (int j = 0; j < S; j++) x[j] = v[j];
    } else
#pragma unroll
        for (int j = 0; j < S; j++) x[j] = S * w + j < N ? row[S * w + j] : 0.0f;
}
template <int S, bool kOnce = false> __device__ __forceinline__ void store_states(float* row, int w, int N, const float* x) {
    if (S == 4 && 4 * w + 4 <= N) {
        four_any4 v;
#pragma unroll
        for (int j = 0; j < S; j++) v[j] = x[j];
        four_any4* at = (four_any4*)(row + 4 * w);
        if (kOnce) __builtin_nontemporal_store(v, at);
        else *at = v;
    } else if (S == 2 && N % 2 == 0 && 2 * w < N) {
        two_any4 v;
#pragma unroll
        for (int j = 0; j < S; j++) v[j] = x[j];
        *(two_any4*)(row + 2 * w) = v;
    } else
#pragma unroll
        for (int j = 0; j < S; j++)
            if (S * w + j < N) row[S * w + j] = x[j];
}
template <int S> __device__ __forceinline__ void clear(float* x) {
#pragma unroll
    for (int j = 0; j < S; j++) x[j] = 0.0f;
}
// S neighbouring numbers of an LDS row
template <int S> __device__ __forceinline__ void read_row(const float* row, float* x) {
    if constexpr (S == 4) {
        const float4 v = *(const float4*)row;
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else if constexpr (S == 2) {
        const float2 v = *(const float2*)row;
        x[0] = v.x, x[1] = v.y;
    } else x[0] = row[0];
}

// h (`from`'s row, or zero) carried over the chunks first .. last - 1 (step +-1)
template <int S, bool kGuard>
__device__ __forceinline__ void fold_over(const ScanArgs& a, int b, int d, int w, int first, int last, int step, const float* A2, const float* from,
                                          float* h) {
    clear<S>(h);
    if (from) load_states<S>(from, w, a.N, h);
#pragma unroll 1                       // eight at a time took the registers of a sixth workgroup per CU
    for (int c = first; c != last; c += step) {
        const long long at = ((long long)b * a.chunks + c) * a.D + d;
        const float sum = a.chunk_dt[at];
        float x[S];
        load_states<S>(a.chunk_h + at * a.N, w, a.N, x);
#pragma unroll
        for (int j = 0; j < S; j++) h[j] = (sum == sum && !(kGuard && h[j] == 0.0f) ? exp2_hw(sum * A2[j]) * h[j] : 0.0f) + x[j];
    }
}
// state (or gradient of a state) that a chunk starts from, folded over the chunks before it.  Where A > 0 a chunk's growth may be beyond the
// type; nothing grows from zero all the same, but inf times 0 is NaN: such a fold is done again with an eye on it (a look at every chunk cost
// 266 -> 283 us at 1 x 16384 x 64, forward and backward).
template <int S>
__device__ __forceinline__ void fold_chunks(const ScanArgs& a, int b, int d, int w, int first, int last, int step, const float* A2, const float* from,
                                            float* h) {
    fold_over<S, false>(a, b, d, w, first, last, step, A2, from, h);
    bool lost = false;
#pragma unroll
    for (int j = 0; j < S; j++) lost |= h[j] != h[j];
    AG_RARE(lost) fold_over<S, true>(a, b, d, w, first, last, step, A2, from, h);
}

// kStates: the first pass over chunks (every chunk but the last; no outputs but chunk_h and chunk_dt).  Otherwise the scan itself.
// A workgroup takes every `rows`-th sequence; while a tile is worked on, the next one's inputs - of the same sequence or the next - are
// on their way.
template <typename T, int NG, int S, bool kStates>
__global__ __launch_bounds__(kLanes* NG, 6) void scan_fwd_kernel(ScanArgs a) {
    constexpr int kRows = kTile / NG, kWide = S * NG;
    __shared__ float2 sdt[kTile][kLanes];                               // dt, dt u
    __shared__ float sy[kStates ? 1 : NG][kTile][kLanes];
    __shared__ alignas(16) float sB[kTile][kWide], sC[kTile][kWide];
    const Place p = place_of(a);
    const int lane = p.lane, w = p.w, d = p.d, N = a.N, T_ = a.T, D = a.D;
    if (kStates && p.chunk == a.chunks - 1) return;
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;
    const bool gate = !kStates && a.z, soft = a.softplus, ckpt = !kStates && a.ckpt;
    const Range mine = chunk_of(a, p);
    const int from = mine.from, to = mine.to;

    float A2[S];
    load_states<S>(a.A + (long long)d * N, w, N, A2);
#pragma unroll
    for (int j = 0; j < S; j++) A2[j] *= kLog2e;
    const int brow = threadIdx.x / kWide, bn = threadIdx.x % kWide;
    const unsigned at = (unsigned)d * (unsigned)sizeof(T);
    const long long state = (long long)d * N;                          // of the lane's channel
    const bool flagged = a.resets;
    Rows u, delta, z, Bm, Cm;
    T ru[kRows] = {}, rd[kRows] = {}, rz[kRows] = {}, rB, rC;
    unsigned char rF = 0;
    auto sequence = [&](int b) __attribute__((always_inline)) {        // its first tile in this chunk
        const auto k = scan_args();
        u.set(k->u, b * k->ub + from * k->ut, k->ut, sizeof(T));
        delta.set(k->delta, b * k->db + from * k->dt, k->dt, sizeof(T));
        if (gate) z.set(k->z, b * k->zb + from * k->zt, k->zt, sizeof(T));
        Bm.set(k->Bm, b * k->bb + p.g * k->bg + from * k->bt, k->bt, sizeof(T));
        if (!kStates) Cm.set(k->Cm, b * k->cb + p.g * k->cg + from * k->ct, k->ct, sizeof(T));
    };
    // a tile's rows, as they are stored; then on to the next tile's
    auto load = [&](int b, int t0, int nv) __attribute__((always_inline)) {
        if (flagged) rF = reset_flag(scan_args(), b, t0, min(nv, kTile), lane);
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int r = w + k * NG;
            if (r < nv) {
                ru[k] = get<T>(u, r, at);
                rd[k] = get<T>(delta, r, at);
                if (gate) rz[k] = get<T>(z, r, at);
            }
        }
        rB = rC = from_f32<T>(0.0f);
        if ((S == 4 || brow < kTile) && brow < nv && bn < N) {
            rB = get<T>(Bm, brow, bn * (unsigned)sizeof(T));
            if (!kStates) rC = get<T>(Cm, brow, bn * (unsigned)sizeof(T));
        }
        u.move(kTile), delta.move(kTile), Bm.move(kTile);
        if (gate) z.move(kTile);
        if (!kStates) Cm.move(kTile);
    };
    int loaded = -1;                                                    // sequence whose first tile is on its way
    float total = 0.0f;                                                 // kStates: sum of dt over the rows this wave staged
    bool any_cut = false;
    for (int b = p.row; b < a.B; b += a.rows) {
        const auto k1 = scan_args();
        const int len = seq_len(k1->lengths, b, T_), end = min(to, len);
        char* out = (char*)k1->out + ((long long)b * T_ + from) * D * (long long)sizeof(T);
        float* ck = k1->ckpt + ((long long)b * ((T_ - 1) / kBack) + from / kBack - 1) * D * N + state;
        if (from < end && loaded != b) {
            sequence(b);
            load(b, from, end - from);
        }
        float h[S];
        clear<S>(h);
        if (!kStates) {
            const float* s0 = k1->s0 ? k1->s0 + (long long)b * D * N + state : nullptr;
            if (p.chunk && from < end) fold_chunks<S>(a, b, d, w, 0, p.chunk, 1, A2, s0, h);
            else if (s0) load_states<S>(s0, w, N, h);
        }
        for (int t0 = from; t0 < end; t0 += kTile) {
            const int nv = min(kTile, end - t0);
            float dt[kRows], uu[kRows], zz[kRows];
#pragma unroll
            for (int k = 0; k < kRows; k++) dt[k] = to_f32(rd[k]) + bias;
            if (soft)
#pragma unroll
                for (int k = 0; k < kRows; k++) dt[k] = softplus(dt[k]);
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const int r = w + k * NG;
                dt[k] = r < nv ? dt[k] : 0.0f;                          // (a row that was not loaded holds an older one)
                uu[k] = r < nv ? to_f32(ru[k]) : 0.0f;
                zz[k] = to_f32(rz[k]);
                if (kStates) total += dt[k];
                sdt[r][lane] = make_float2(dt[k], dt[k] * uu[k]);
            }
            if (S == 4 || brow < kTile) {
                sB[brow][bn] = to_f32(rB);
                if (!kStates) sC[brow][bn] = to_f32(rC);
            }
            const unsigned cut = reset_bits(rF);
            any_cut |= cut != 0;
            __syncthreads();
            int next = end - t0 - kTile, next_b = b, next_t = t0 + kTile;
            if (!kStates && next <= 0 && b + a.rows < a.B) {
                loaded = next_b = b + a.rows;
                next_t = from;
                sequence(next_b);
                next = min(to, seq_len(scan_args()->lengths, next_b, T_)) - from;
            }
            if (next > 0) load(next_b, next_t, next);
#pragma unroll
            for (int r = 0; r < kTile; r++) {                           // steps behind nv have dt = 0: they change nothing
                if (r % 4 == 0 && r >= nv) break;
                if (r % kBack == 0 && ckpt) {
                    if (t0 + r && p.live) store_states<S>(ck, w, N, h);
                    ck += (long long)D * N;
                }
                AG_RARE(cut >> r & 1) clear<S>(h);
                const float2 q = sdt[r][lane];
                float Bn[S], Cn[S], y = 0.0f;
                read_row<S>(&sB[r][S * w], Bn);
                if (!kStates) read_row<S>(&sC[r][S * w], Cn);
#pragma unroll
                for (int j = 0; j < S; j++) {
                    h[j] = __builtin_fmaf(exp2_hw(q.x * A2[j]), h[j], q.y * Bn[j]);
                    if (!kStates) y = j ? __builtin_fmaf(Cn[j], h[j], y) : Cn[j] * h[j];
                }
                if (!kStates) sy[w][r][lane] = y;
            }
            __syncthreads();
            if (!kStates) {
                float y[kRows];
#pragma unroll
                for (int k = 0; k < kRows; k++) {
                    y[k] = skip * uu[k];
#pragma unroll
                    for (int v = 0; v < NG; v++) y[k] += sy[v][w + k * NG][lane];      // (rows behind nv: whatever is there, not stored)
                }
                if (gate)
#pragma unroll
                    for (int k = 0; k < kRows; k++) y[k] *= zz[k] * sigmoid(zz[k]);
#pragma unroll
                for (int k = 0; k < kRows; k++) {
                    const int r = w + k * NG;
                    if (r < nv && p.live) put(out, r * (D * (unsigned)sizeof(T)) + at, from_f32<T>(y[k]));
                }
                out += (long long)kTile * D * (long long)sizeof(T);
            }
        }
        const auto k2 = scan_args();
        if (kStates) {
            float* sums = (float*)sdt;
            sums[w * kLanes + lane] = total;
            __syncthreads();
            if (!p.live) return;
            const long long row = ((long long)b * a.chunks + p.chunk) * D + d;
            store_states<S>(k2->chunk_h + row * N, w, N, h);
            if (w == 0) {
                float s = 0.0f;
                for (int v = 0; v < NG; v++) s += sums[v * kLanes + lane];
                k2->chunk_dt[row] = any_cut ? __builtin_nanf("") : s;
            }
            return;                                                     // chunks: one sequence per workgroup
        }
        if (!p.live) continue;
        if (len < T_) {
            out = (char*)k2->out + (long long)b * T_ * D * (long long)sizeof(T);
            const Range pad = padding_of(k2, p, len);
            for (int t = pad.from + w; t < pad.to; t += NG) put(out + (long long)t * D * (long long)sizeof(T), at, from_f32<T>(0.0f));
        }
        if (k2->s1 && (len ? from < len && len <= to : p.chunk == 0))   // the chunk with the last step
            store_states<S>(k2->s1 + (long long)b * D * N + state, w, N, h);
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
// The states of a tile of 8 steps are run again from the state the forward left before it and kept, with the decays, in registers;
// tiles are walked backwards.  16 steps per tile took 326 registers (one wave per SIMD) and five times as long.  A workgroup takes
// every `rows`-th sequence, so that dA, dD and the bias gradient stay in registers meanwhile.
// dB and dC are sums over channels, that is over lanes: eight values (8 / S steps') at a time, transposed on the way.

// kCarry: the first pass over chunks (every chunk but the first): what the chunk hands back to the one before when nothing reaches it
// from behind, and its sum of dt.
template <typename T, int NG, int S, bool kCarry>
__global__ __launch_bounds__(kLanes* NG, kCarry ? 1 : 3) void scan_bwd_kernel(ScanArgs a, ScanGradArgs q) {
    constexpr int kRows = kBack / NG, kWide = S * NG, kSteps = 8 / S;
    __shared__ float2 sdt[kBack][kLanes];                               // dt, dt u
    __shared__ float sdy[kBack][kLanes];
    __shared__ float skeep[3][kCarry ? 1 : kBack][kLanes];              // u, softplus' slope, what turns y into the gate's gradient
    __shared__ float sy[kCarry ? 1 : NG][kBack][kLanes], ss1[kCarry ? 1 : NG][kBack][kLanes], ss2[kCarry ? 1 : NG][kBack][kLanes];
    __shared__ alignas(16) float sBC[2][kBack][kWide], sdBC[2][kBack][kWide];
    const Place p = place_of(a);
    if (kCarry && p.chunk == 0) return;
    const int lane = p.lane, w = p.w, d = p.d, N = a.N, T_ = a.T, D = a.D;
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;
    const bool gate = a.z, soft = a.softplus;
    const Range own = chunk_of(a, p);
    const int from = own.from, to = own.to, last = to > from ? from + (to - from - 1) / kBack * kBack : from - kBack;      // of its tiles
    // 8 rows of B and of C: a thread has one of each, or none
    const int brow = threadIdx.x / kWide, bn = threadIdx.x % kWide;
    const unsigned at = (unsigned)d * (unsigned)sizeof(T);
    const long long state = (long long)d * N;
    const int GN = a.G * N;
    const unsigned bc_at = brow * GN + p.g * N + bn;                    // in a tile of [T, G, N]
    float A2[S], dA[S], dD = 0.0f, dbias = 0.0f;
    load_states<S>(a.A + state, w, N, A2);
    clear<S>(dA);
#pragma unroll
    for (int j = 0; j < S; j++) A2[j] *= kLog2e;

    const bool flagged = a.resets;
    Rows u, delta, z, dout, Bm, Cm;
    T ru[kRows] = {}, rd[kRows] = {}, rz[kRows] = {}, rg[kRows] = {}, rB, rC;
    unsigned char rF = 0;
    float start[S];
    auto sequence = [&](int b) __attribute__((always_inline)) {        // its last tile in this chunk
        const auto k = scan_args();
        const auto g = grad_args();
        if (!kCarry) u.set(k->u, b * k->ub + last * k->ut, k->ut, sizeof(T));
        delta.set(k->delta, b * k->db + last * k->dt, k->dt, sizeof(T));
        if (gate) z.set(k->z, b * k->zb + last * k->zt, k->zt, sizeof(T));
        dout.set(g->dout, b * g->ob + last * g->ot, g->ot, sizeof(T));
        if (!kCarry) Bm.set(k->Bm, b * k->bb + p.g * k->bg + last * k->bt, k->bt, sizeof(T));
        Cm.set(k->Cm, b * k->cb + p.g * k->cg + last * k->ct, k->ct, sizeof(T));
    };
    // a tile's inputs as they are stored, and the state it starts from (nv <= 0: nothing); then on to the tile before
    auto load = [&](int b, int t0, int nv) __attribute__((always_inline)) {
        if (flagged) rF = reset_flag(scan_args(), b, t0, min(nv, kBack), lane);
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const int r = w + k * NG;
            if (r < nv) {
                if (!kCarry) ru[k] = get<T>(u, r, at);
                rd[k] = get<T>(delta, r, at);
                rg[k] = get<T>(dout, r, at);
                if (gate) rz[k] = get<T>(z, r, at);
            }
        }
        rB = rC = from_f32<T>(0.0f);
        if (brow < kBack && brow < nv && bn < N) {
            if (!kCarry) rB = get<T>(Bm, brow, bn * (unsigned)sizeof(T));
            rC = get<T>(Cm, brow, bn * (unsigned)sizeof(T));
        }
        if (!kCarry && nv > 0) {
            const auto k = scan_args();
            if (t0) load_states<S>(k->ckpt + ((long long)b * ((T_ - 1) / kBack) + t0 / kBack - 1) * D * N + state, w, N, start);
            else if (k->s0) load_states<S>(k->s0 + (long long)b * D * N + state, w, N, start);
            else clear<S>(start);
        }
        if (!kCarry) u.move(-kBack), Bm.move(-kBack);
        delta.move(-kBack), dout.move(-kBack), Cm.move(-kBack);
        if (gate) z.move(-kBack);
    };
    int len = 0;
    if (p.row < a.B) {
        len = seq_len(a.lengths, p.row, T_);
        if (to > from) {
            sequence(p.row);
            load(p.row, last, len - last);
        }
    }
    for (int b = p.row; b < a.B; b += q.rows) {
        const auto k1 = scan_args();
        const auto g1 = grad_args();
        const long long o = ((long long)b * T_ + last) * D * (long long)sizeof(T);
        char *du = (char*)g1->du + o, *ddelta = (char*)g1->ddelta + o, *dz = (char*)g1->dz + o;
        const int next_b = b + q.rows, next_len = next_b < a.B ? seq_len(k1->lengths, next_b, T_) : 0;
        float carry[S];                                                 // a_{t+1} g_{t+1}
        clear<S>(carry);
        if (!kCarry) {
            const float* ds1 = g1->ds1 && p.live ? g1->ds1 + (long long)b * D * N + state : nullptr;
            if (p.chunk < a.chunks - 1) fold_chunks<S>(a, b, d, w, a.chunks - 1, p.chunk, -1, A2, ds1, carry);
            else if (ds1) load_states<S>(ds1, w, N, carry);
        }
        float total = 0.0f;
        bool any_cut = false;
        for (int t0 = last; t0 >= from; t0 -= kBack) {
            const int nv = max(0, min(kBack, len - t0)), nt = min(kBack, T_ - t0);
            float now[S];
#pragma unroll
            for (int j = 0; j < S; j++) now[j] = p.live ? start[j] : 0.0f;
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const int r = w + k * NG;
                float dt = 0.0f, dy = 0.0f, uu = 0.0f, slope = 0.0f, dg = 0.0f;
                if (r < nv && p.live) {
                    if (!kCarry) uu = to_f32(ru[k]);
                    dt = to_f32(rd[k]) + bias;
                    slope = 1.0f;
                    if (soft) dt = softplus(dt, slope);
                    dy = to_f32(rg[k]);
                    if (gate) {
                        const float zz = to_f32(rz[k]), sz = sigmoid(zz);
                        dg = dy * sz * __builtin_fmaf(zz, 1.0f - sz, 1.0f);
                        dy *= sz * zz;
                    }
                }
                sdt[r][lane] = make_float2(dt, dt * uu);
                sdy[r][lane] = dy;
                if (!kCarry) skeep[0][r][lane] = uu, skeep[1][r][lane] = slope, skeep[2][r][lane] = dg;
                if (kCarry) total += dt;
            }
            if (brow < kBack) {
                if (!kCarry) sBC[0][brow][bn] = to_f32(rB);
                sBC[1][brow][bn] = to_f32(rC);
            }
            const unsigned cut = reset_bits(rF);
            any_cut |= cut != 0;
            __syncthreads();
            const bool same = t0 > from;
            if (!same && next_b < a.B) sequence(next_b);
            load(same ? b : next_b, same ? t0 - kBack : last, same ? len - t0 + kBack : next_len - last);
            if (kCarry) {
                auto back = [&](auto kCut) __attribute__((always_inline)) {
#pragma unroll
                    for (int r = kBack - 1; r >= 0; r--) {
                        const float dy = sdy[r][lane], dt = sdt[r][lane].x;
                        float Cn[S];
                        read_row<S>(&sBC[1][r][S * w], Cn);
#pragma unroll
                        for (int j = 0; j < S; j++) carry[j] = exp2_hw(dt * A2[j]) * __builtin_fmaf(Cn[j], dy, carry[j]);
                        if (kCut.value) keep_if<S>(!(cut >> r & 1), carry);
                    }
                };
                if (cut) back(Flag<true>{});
                else back(Flag<false>{});
                __syncthreads();
                continue;
            }
            auto tile = [&](auto kCut) __attribute__((always_inline)) {
                float h[kBack][S], e[kBack][S], v[8], sums = 0.0f;      // h[r]: the state step r starts from
                // kSteps steps' values are summed at a time; lane 8g + i keeps the i-th sum
                const int order = sum_lanes8_order(lane), step = order / S, mine = lane % S;
#pragma unroll
                for (int r = 0; r < kBack; r++) {      // steps behind nv have dt = dy = 0: decay 1, no input
                    if (kCut.value) keep_if<S>(!(cut >> r & 1), now);
                    const float2 s = sdt[r][lane];
                    const float dy = sdy[r][lane];
                    float Bn[S], Cn[S];
                    read_row<S>(&sBC[0][r][S * w], Bn);
                    read_row<S>(&sBC[1][r][S * w], Cn);
                    float y = 0.0f;
#pragma unroll
                    for (int j = 0; j < S; j++) {
                        h[r][j] = now[j];
                        e[r][j] = exp2_hw(s.x * A2[j]);
                        now[j] = __builtin_fmaf(e[r][j], now[j], s.y * Bn[j]);
                        y = j ? __builtin_fmaf(Cn[j], now[j], y) : Cn[j] * now[j];
                        v[r % kSteps * S + j] = dy * now[j];
                    }
                    sy[w][r][lane] = y;
                    if (r % kSteps == kSteps - 1) {
                        const float x = sum_lanes8(v, lane);
                        sums = mine == r / kSteps ? x : sums;
                    }
                }
                // nothing is moved across: with both passes' reads ahead of the first the kernel keeps 46 registers in memory (780 us
                // where it takes 426)
                __builtin_amdgcn_sched_barrier(0);
                if ((lane & 7) < S) sdBC[1][kSteps * mine + step][S * w + order % S] = sums;
#pragma unroll
                for (int r = kBack - 1; r >= 0; r--) {
                    const float2 s = sdt[r][lane];
                    const float dy = sdy[r][lane];
                    float Bn[S], Cn[S];
                    read_row<S>(&sBC[0][r][S * w], Bn);
                    read_row<S>(&sBC[1][r][S * w], Cn);
                    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
                    for (int j = 0; j < S; j++) {
                        const float gr = __builtin_fmaf(Cn[j], dy, carry[j]);
                        v[r % kSteps * S + j] = gr * s.y;
                        s1 = j ? __builtin_fmaf(gr, Bn[j], s1) : gr * Bn[j];
                        carry[j] = e[r][j] * gr;
                        const float qq = carry[j] * h[r][j];
                        s2 = j ? __builtin_fmaf(qq, A2[j], s2) : qq * A2[j];
                        dA[j] = __builtin_fmaf(qq, s.x, dA[j]);
                    }
                    if (kCut.value) keep_if<S>(!(cut >> r & 1), carry);     // h[r] is 0 there already
                    ss1[w][r][lane] = s1;
                    ss2[w][r][lane] = s2;
                    if (r % kSteps == 0) {
                        const float x = sum_lanes8(v, lane);
                        sums = mine == r / kSteps ? x : sums;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if ((lane & 7) < S) sdBC[0][kSteps * mine + step][S * w + order % S] = sums;
            };
            if (nv) {
                if (cut) tile(Flag<true>{});
                else tile(Flag<false>{});
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const int r = w + k * NG;
                if (r >= nt) break;
                const float uu = skeep[0][r][lane];
                float y = skip * uu, s1 = 0.0f, s2 = 0.0f;
                if (r < nv) {
#pragma unroll
                    for (int v = 0; v < NG; v++) y += sy[v][r][lane], s1 += ss1[v][r][lane], s2 += ss2[v][r][lane];
                }
                const float dy = sdy[r][lane], dt = sdt[r][lane].x;
                const float draw = __builtin_fmaf(uu, s1, s2 * kLn2) * skeep[1][r][lane];      // s2 was summed with A log2(e)
                if (p.live) {
                    const unsigned i = r * (D * (unsigned)sizeof(T)) + at;
                    put(du, i, from_f32<T>(__builtin_fmaf(dt, s1, skip * dy)));
                    put(ddelta, i, from_f32<T>(draw));
                    if (gate) put(dz, i, from_f32<T>(skeep[2][r][lane] * y));
                }
                dD = __builtin_fmaf(dy, uu, dD);
                dbias += draw;
            }
            const long long back = (long long)kBack * D * (long long)sizeof(T);
            du -= back, ddelta -= back, dz -= back;
            if (brow < nt && bn < N) {                                  // nt <= 8
                const auto g = grad_args();
                const float vB = brow < nv ? sdBC[0][brow][bn] : 0.0f, vC = brow < nv ? sdBC[1][brow][bn] : 0.0f;
                const long long first = ((long long)b * T_ + t0) * GN;
                if (g->bc_partials) {
                    const long long all = (long long)a.B * T_ * GN;
                    float* part = g->bc_partials + (2 * p.cb * all + first);
                    part[bc_at] = vB;
                    (part + all)[bc_at] = vC;
                } else {
                    ((T*)g->dB + first)[bc_at] = from_f32<T>(vB);
                    ((T*)g->dC + first)[bc_at] = from_f32<T>(vC);
                }
            }
        }
        if (!kCarry && a.chunks > 1 && len < T_) {                      // (without chunks the tiles behind the end have written theirs)
            const auto k = scan_args();
            const auto g = grad_args();
            const Range pad = padding_of(k, p, (len + kBack - 1) / kBack * kBack);
            const long long row = (long long)b * T_;
            for (int t = pad.from + w; p.live && t < pad.to; t += NG) {
                const long long bytes = (row + t) * D * (long long)sizeof(T);
                put((char*)g->du + bytes, at, from_f32<T>(0.0f));
                put((char*)g->ddelta + bytes, at, from_f32<T>(0.0f));
                if (gate) put((char*)g->dz + bytes, at, from_f32<T>(0.0f));
            }
            for (int t = pad.from + brow; bn < N && t < pad.to; t += kLanes / S) {
                const long long i = (row + t) * GN + p.g * N + bn, all = (long long)k->B * T_ * GN;
                if (g->bc_partials) {
                    float* part = g->bc_partials + 2 * p.cb * all + i;
                    part[0] = part[all] = 0.0f;
                } else ((T*)g->dB)[i] = ((T*)g->dC)[i] = from_f32<T>(0.0f);
            }
        }
        len = next_len;
        const auto k2 = scan_args();
        const auto g2 = grad_args();
        if (kCarry) {
            float* sums = (float*)sdt;
            sums[w * kLanes + lane] = total;
            __syncthreads();
            if (p.live) {
                const long long row = ((long long)b * k2->chunks + p.chunk) * D + d;
                store_states<S>(k2->chunk_h + row * N, w, N, carry);
                if (w == 0) {
                    float s = 0.0f;
                    for (int v = 0; v < NG; v++) s += sums[v * kLanes + lane];
                    k2->chunk_dt[row] = any_cut ? __builtin_nanf("") : s;
                }
            }
            __syncthreads();
        } else if (g2->ds0 && p.live && p.chunk == 0)
            store_states<S>(g2->ds0 + (long long)b * D * N + state, w, N, carry);
    }
    if (kCarry) return;
    // this workgroup's row of partial parameter gradients: [rows chunks, D, N + 2]
    float* part = grad_args()->param_partials + ((long long)(p.row * a.chunks + p.chunk) * D + d) * (N + 2);
    __syncthreads();
    float2* sums = &sdt[0][0];
    sums[w * kLanes + lane] = make_float2(dD, dbias);
    __syncthreads();
    if (!p.live) return;
#pragma unroll
    for (int j = 0; j < S; j++)
        if (S * w + j < N) part[S * w + j] = dA[j];
    if (w == 0) {
        float s = 0.0f, t = 0.0f;
#pragma unroll
        for (int v = 0; v < NG; v++) s += sums[v * kLanes + lane].x, t += sums[v * kLanes + lane].y;
        part[N] = s;
        part[N + 1] = t;
    }
}

struct ScanParams {
    float *dA, *dD, *dbias;
    int N;
    __device__ __forceinline__ void operator()(long long i, float s) const {
        const long long d = i / (N + 2);
        const int k = (int)(i - d * (N + 2));
        if (k < N) dA[d * N + k] = s;
        else if (k == N) { if (dD) dD[d] = s; }
        else if (dbias) dbias[d] = s;
    }
};

template <typename T> struct ScanShared {
    T *dB, *dC;
    long long n;
    __device__ __forceinline__ void operator()(long long i, float s) const {
        if (i < n) dB[i] = from_f32<T>(s);
        else dC[i - n] = from_f32<T>(s);
    }
};

// One step: a channel's state is spread over L lanes, four numbers each, so that a wave moves 1 KB of states per access; the states
// in and out are nearly all of the bytes, each touched once.
// kShared: a wave takes up to 64 channels of one sequence and group.  Each lane then also owns one of the channels and forms its time
// step and its gate, the L rounds over the states fetch them from there, B and C are read once for all of them, and L accesses per lane
// are in flight.  Otherwise a wave's 64 / L channels lie anywhere.  kTail: N is above 4 and no multiple of it.
// Bytes bound it: 4096 x 512, N = 16, float32 takes 52 us = 5.8 TB/s, bfloat16 52 us = 5.4 TB/s (an in-place product over the states
// alone 48 us).  Large states are marked as used once (the rule and both sides stand where it is chosen); without sharing the float32 step
// took 61 us.
template <typename T, int L, bool kShared, bool kTail, bool kOnce>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
    constexpr int kRounds = kShared ? L : 1, C = 64 / L;                  // channels of a wave per round
    const int l = threadIdx.x & 63, part = l % L, mine = kShared ? l / L : 0;        // the lane's channel behind c0 in round 0
    const unsigned wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), D = a.D;
    unsigned b, c0, d, g, end;                                            // B D < 2^31
    if (kShared) {
        const unsigned per = (unsigned)a.nb * (unsigned)a.G, in = wave % per;
        b = wave / per, g = in / (unsigned)a.nb;
        c0 = g * (unsigned)a.Dg + in % (unsigned)a.nb * 64, end = (g + 1) * (unsigned)a.Dg, d = min(c0 + l, end - 1);
    } else {
        const unsigned item = wave * C + l / L;
        b = item / D, d = c0 = item % D, end = D, g = a.G > 1 ? d / (unsigned)a.Dg : 0;
    }
    if (b >= (unsigned)a.B) return;
    const long long row = (long long)b * D + c0;
    float h[kRounds][4], A[kRounds][4], Bn[4], Cn[4];
#pragma unroll
    for (int i = 0; i < kRounds; i++) {
        clear<4>(h[i]);
        if (a.s0 && c0 + i * C + mine < end) load_states<4, kOnce, kTail>(a.s0 + (row + i * C + mine) * a.N, part, a.N, h[i]);
    }
    const T* Bm = (const T*)a.Bm + (b * a.bb + g * a.bg);
    const T* Cm = (const T*)a.Cm + (b * a.cb + g * a.cg);
    const bool cut = a.resets && a.resets[b * a.rb];
    const float u = to_f32(((const T*)a.u)[b * a.ub + d]), raw = to_f32(((const T*)a.delta)[b * a.db + d]);
    const float z = a.z ? to_f32(((const T*)a.z)[b * a.zb + d]) : 0.0f;
    clear<4>(Bn), clear<4>(Cn);
    if (kTail || a.N % 4 == 0) {
        const int from = min(4 * part, a.N - 4);
        const auto vB = load_vec<T, 4>(Bm + from), vC = load_vec<T, 4>(Cm + from);
        const float cB[4] = {vB.at(0), vB.at(1), vB.at(2), vB.at(3)}, cC[4] = {vC.at(0), vC.at(1), vC.at(2), vC.at(3)};
        if (kTail) shift_down(cB, 4 * part - from, Bn), shift_down(cC, 4 * part - from, Cn);
        else if (4 * part < a.N)
#pragma unroll
            for (int j = 0; j < 4; j++) Bn[j] = cB[j], Cn[j] = cC[j];
    } else
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (4 * part + j < a.N) Bn[j] = to_f32(Bm[4 * part + j]), Cn[j] = to_f32(Cm[4 * part + j]);
#pragma unroll
    for (int i = 0; i < kRounds; i++) load_states<4, false, kTail>(a.A + (long long)min(c0 + i * C + mine, end - 1) * a.N, part, a.N, A[i]);
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;
    const float dt = a.softplus ? softplus(raw + bias) : raw + bias, dtu = dt * u;
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < kRounds; i++) {
        const bool fetch = kShared && L > 1;
        const float t = fetch ? __shfl(dt, i * C + mine) : dt, tu = fetch ? __shfl(dtu, i * C + mine) : dtu;
        float p = 0.0f;
        if (cut) clear<4>(h[i]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            h[i][j] = __builtin_fmaf(exp2_hw(t * (A[i][j] * kLog2e)), h[i][j], tu * Bn[j]);
            p = __builtin_fmaf(Cn[j], h[i][j], p);
        }
        if (c0 + i * C + mine < end) store_states<4, kOnce>(a.s1 + (row + i * C + mine) * a.N, part, a.N, h[i]);
        if (L > 1) p += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(p), 0xB1, 0xf, 0xf, true));
        if (L > 2) p += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(p), 0x4E, 0xf, 0xf, true));
        if (L > 4) p += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(p), 0x141, 0xf, 0xf, true));
        const float q = fetch ? __shfl(p, l % C * L) : p;                 // a round's channels are its lanes L, 2 L, ...
        y = !kShared || l / C == i ? q : y;
    }
    float o = __builtin_fmaf(skip, u, y);
    if (a.z) o *= z * sigmoid(z);
    if (kShared ? c0 + l < end : part == 0) ((T*)a.out)[(long long)b * D + d] = from_f32<T>(o);
}

int step_lanes(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8; }
int channel_blocks(int D, int G) { return (D / G + kLanes - 1) / kLanes; }

// Chunks of time.  1536 workgroups are six per CU, what the forward's registers let in and two rounds of the backward; where sequences
// and channels give fewer, time is cut so that there are about that many, in chunks of at least 64 steps (a multiple of 16).  Forward and
// backward in bf16 with 768, 1024, 1536, 2304 and twice 1536 workgroups: 785, 722, 657, 652 and 646 us at B = 8, T = 2047, D = 2048 with lengths
// drawn evenly; 864, 914, 833, 857 and 853 in full length; 263, 268, 279, 291 and 290 at B = 1, T = 4096, where each chunk has more chunks
// before it to start from.
int chunks_of(int B, int T, int D, int G) {
    const long long blocks = (long long)B * G * channel_blocks(D, G);
    const long long want = (1536 + blocks - 1) / blocks;
    long long steps = ((T + want - 1) / want + kTile - 1) / kTile * kTile;
    if (steps < 64) steps = 64;
    return want == 1 || steps >= T ? 1 : (int)((T + steps - 1) / steps);
}

// workgroups along the batch, each of which takes several sequences where there are many: two rounds of what the CUs hold (forward
// six workgroups per CU, backward three)
int rows_of(int B, int D, int G, int resident) {
    const int per = channel_blocks(D, G) * G, want = (2 * 256 * resident + per - 1) / per;
    return B < want ? B : want;
}
int grad_rows(int B, int D, int G) { return rows_of(B, D, G, 3); }

int check(const ag_scan_args* p) {
    if (!p || p->struct_size != sizeof(ag_scan_args) || !p->u_dev || !p->delta_dev || !p->Bm_dev || !p->Cm_dev || !p->A_dev)
        return AG_ERR_INVALID_ARG;
    if (p->B <= 0 || p->T <= 0 || p->D <= 0 || p->G <= 0 || p->N <= 0 || p->D % p->G) return AG_ERR_INVALID_ARG;
    if (p->N > 32 || p->dtype < AG_F32 || p->dtype > AG_F16) return AG_ERR_UNSUPPORTED;
    if (p->u_st < 0 || p->delta_st < 0 || p->z_st < 0 || p->b_st < 0 || p->c_st < 0) return AG_ERR_INVALID_ARG;
    // a lane's offset within a tile's rows has 32 bits
    const long long most = (0xffffffffLL / 4 - p->D) / kTile;
    if (p->D > most || p->u_st > most || p->delta_st > most || p->z_st > most || p->b_st > most || p->c_st > most) return AG_ERR_UNSUPPORTED;
    // the grid: rows_of or chunks_of make it some thousands of workgroups of up to 512 threads, but one per block of channels at least;
    // with it G N (at most 32 G) times a tile's steps stays within 32 bits
    if (p->T > kMaxSteps || (long long)p->G * channel_blocks(p->D, p->G) > 1 << 21) return AG_ERR_UNSUPPORTED;
    return AG_OK;
}

ScanArgs device_args(const ag_scan_args* p) {
    const int chunks = chunks_of(p->B, p->T, p->D, p->G);
    return ScanArgs{p->u_dev, p->delta_dev, p->z_dev, p->Bm_dev, p->Cm_dev, p->A_dev, p->Dskip_dev, p->delta_bias_dev, p->state_in_dev,
                    p->lengths_dev, p->resets_dev, p->u_sb, p->u_st, p->delta_sb, p->delta_st, p->z_sb, p->z_st, p->b_sb, p->b_st, p->b_sg,
                    p->c_sb, p->c_st, p->c_sg, p->r_sb, p->r_st, p->out_dev, p->state_out_dev, p->ckpt_dev, nullptr, nullptr, p->B, p->T,
                    p->D, p->N, p->G, p->softplus, p->D / p->G, channel_blocks(p->D, p->G),
                    chunks > 1 ? p->B : rows_of(p->B, p->D, p->G, 6), chunks};
}

// floats of chunk_h and chunk_dt
long long chunk_floats(int B, int T, int D, int N, int G) {
    const int c = chunks_of(B, T, D, G);
    return c > 1 ? (long long)B * c * D * (N + 1) : 0;
}

}  // namespace

// Four waves up to 16 states, eight beyond; 1, 2 or 4 states per lane.  (One or two waves of four states a lane for N <= 8 would have to
// stage all rows themselves: 4096 x 24 x 256 f32, forward and backward, took 523 and 533 us at N = 8 and 4 against 601 at N = 16.)
#define AG_FOR_STATES(N_, CALL)                                                  \
    do {                                                                         \
        if (N_ <= 4) { constexpr int NG = 4, S = 1; CALL; }                      \
        else if (N_ <= 8) { constexpr int NG = 4, S = 2; CALL; }                 \
        else if (N_ <= 16) { constexpr int NG = 4, S = 4; CALL; }                \
        else { constexpr int NG = 8, S = 4; CALL; }                              \
    } while (0)

#define AG_FOR_LANES(N_, CALL)                                                   \
    do {                                                                         \
        switch (step_lanes(N_)) {                                                \
            case 1: { constexpr int L = 1; CALL; } break;                        \
            case 2: { constexpr int L = 2; CALL; } break;                        \
            case 4: { constexpr int L = 4; CALL; } break;                        \
            default: { constexpr int L = 8; CALL; } break;                       \
        }                                                                        \
    } while (0)

extern "C" long long ag_selective_scan_ckpt_floats(int B, int T, int D, int N) {
    if (B <= 0 || T <= 0 || D <= 0 || N <= 0) return 0;
    return (long long)B * ((T - 1) / kBack) * D * N;
}

extern "C" long long ag_selective_scan_workspace_bytes(int B, int T, int D, int N, int G, int backward) {
    if (B <= 0 || T <= 0 || D <= 0 || N <= 0 || G <= 0 || D % G) return 0;
    long long floats = chunk_floats(B, T, D, N, G);
    if (backward) {
        const int nb = channel_blocks(D, G);
        floats += (long long)grad_rows(B, D, G) * chunks_of(B, T, D, G) * D * (N + 2);
        if (nb > 1) floats += 2LL * nb * B * T * G * N;
    }
    return floats * (long long)sizeof(float);
}

extern "C" int ag_selective_scan_fwd(const ag_scan_args* p, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!p->out_dev) return AG_ERR_INVALID_ARG;
    ScanArgs a = device_args(p);
    if (a.chunks > 1) {
        if (!p->workspace_dev || p->workspace_bytes < ag_selective_scan_workspace_bytes(a.B, a.T, a.D, a.N, a.G, 0)) return AG_ERR_INVALID_ARG;
        a.chunk_h = (float*)p->workspace_dev;
        a.chunk_dt = a.chunk_h + (long long)a.B * a.chunks * a.D * a.N;
    }
    const dim3 grid((unsigned)((long long)a.rows * a.chunks * a.G * a.nb));
    if (a.chunks > 1)
        AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_fwd_kernel<T, NG, S, true>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a)));
    AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_fwd_kernel<T, NG, S, false>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a)));
    return seq_status();
}

extern "C" int ag_selective_scan_bwd(const ag_scan_args* p, const ag_scan_grads* r, void* stream) {
    if (const int rc = check(p)) return rc;
    if (!r || r->struct_size != sizeof(ag_scan_grads) || !r->dout_dev || !r->du_dev || !r->ddelta_dev || !r->dBm_dev || !r->dCm_dev ||
        !r->dA_dev || !r->workspace_dev || (p->z_dev != nullptr) != (r->dz_dev != nullptr) || (p->T > kBack && !p->ckpt_dev))
        return AG_ERR_INVALID_ARG;
    if (r->workspace_bytes < ag_selective_scan_workspace_bytes(p->B, p->T, p->D, p->N, p->G, 1)) return AG_ERR_INVALID_ARG;
    if (r->dout_st < 0) return AG_ERR_INVALID_ARG;
    if (r->dout_st > (0xffffffffLL / 4 - p->D) / kTile) return AG_ERR_UNSUPPORTED;
    ScanArgs a = device_args(p);
    a.chunk_h = (float*)r->workspace_dev;
    a.chunk_dt = a.chunk_h + (long long)a.B * a.chunks * a.D * a.N;
    float* params = a.chunk_h + chunk_floats(a.B, a.T, a.D, a.N, a.G);
    const int rows = grad_rows(a.B, a.D, a.G);
    float* bc = a.nb > 1 ? params + (long long)rows * a.chunks * a.D * (a.N + 2) : nullptr;
    const ScanGradArgs q{r->dout_dev, r->dout_sb, r->dout_st, r->dstate_out_dev, r->du_dev, r->ddelta_dev, r->dz_dev, r->dBm_dev, r->dCm_dev,
                         r->dstate_in_dev, params, bc, rows};
    const dim3 grid((unsigned)((long long)rows * a.chunks * a.G * a.nb));
    if (a.chunks > 1)
        AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_bwd_kernel<T, NG, S, true>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a, q)));
    AG_FOR_DTYPE(p->dtype, AG_FOR_STATES(p->N, hipLaunchKernelGGL((scan_bwd_kernel<T, NG, S, false>), grid, dim3(kLanes * NG), 0, (hipStream_t)stream, a, q)));
    launch_sum_rows(params, rows * a.chunks, (long long)a.D * (a.N + 2), ScanParams{r->dA_dev, r->dDskip_dev, r->ddelta_bias_dev, a.N}, stream);
    if (bc) {
        const long long n = (long long)a.B * a.T * a.G * a.N;
        AG_FOR_DTYPE(p->dtype, launch_sum_rows(bc, a.nb, 2 * n, ScanShared<T>{(T*)r->dBm_dev, (T*)r->dCm_dev, n}, stream));
    }
    return seq_status();
}

extern "C" int ag_selective_scan_step(const ag_scan_args* p, void* stream) {
    if (const int rc = check(p)) return rc;
    if (p->T != 1 || !p->out_dev || !p->state_out_dev) return AG_ERR_INVALID_ARG;
    const ScanArgs a = device_args(p);
    const int lanes = step_lanes(p->N);
    if ((long long)a.B * a.D > 0x7fffffffLL) return AG_ERR_UNSUPPORTED;
    // where the channels of a group fill the lanes of its waves to four fifths and more (4096 x 512 in 16 groups of 32 channels: 69 us
    // not shared; 4096 x 500: 53 us shared, 69 us not)
    const bool shared = a.nb * 64LL * 4 <= a.Dg * 5LL, tail = a.N > 4 && a.N % 4;
    const long long waves = shared ? (long long)a.B * a.G * a.nb : ((long long)a.B * a.D * lanes + 63) / 64, blocks = (waves + 3) / 4;
    if (blocks > kMaxThreads / 256) return AG_ERR_UNSUPPORTED;
    // From half of the last-level cache on a state is marked as used once.  One state moved on again and again, with nothing between the steps,
    // pays for it; a state that other work has driven out (here: three batches in turn) gains.  Plain and marked, in us, at N = 16, D = 512:
    //   float32   64 MiB 27.6, 27.6 and 27.1, 28.8    128 MiB 49.7, 52 and 63.3, 52    192 MiB 72.0, 74.5 and 90.3, 74.5    256 MiB 107, 97 and 117, 97
    //   bfloat16  64 MiB 28.1, 25.8 and 27.6, 27.4    128 MiB 49.3, 49.8 and 60.8, 50.8    256 MiB 98, 95 and 112, 95
    const bool once = (long long)a.B * a.D * a.N * 4 >= kCached;
    const dim3 grid((unsigned)blocks), block(256);
#define AG_STEP(SHARED, TAIL, ONCE)                                                                                              \
    AG_FOR_DTYPE(p->dtype, AG_FOR_LANES(p->N, hipLaunchKernelGGL((scan_step_kernel<T, L, SHARED, (TAIL && L > 1), ONCE>), grid, block, 0, \
                                                                 (hipStream_t)stream, a)))
    if (shared && tail && once) AG_STEP(true, true, true);
    else if (shared && tail) AG_STEP(true, true, false);
    else if (shared && once) AG_STEP(true, false, true);
    else if (shared) AG_STEP(true, false, false);
    else if (tail && once) AG_STEP(false, true, true);
    else if (tail) AG_STEP(false, true, false);
    else if (once) AG_STEP(false, false, true);
    else AG_STEP(false, false, false);
#undef AG_STEP
    return seq_status();
}
