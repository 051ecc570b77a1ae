// Norms before and after a block of a sequence model, with the gate, the residual scale, the residual and the norm in
// front of the next block in the same pass, and their gradients (pathsig_norm_* of pathsig_hip.h).
//
// Forward, for a row x of C channels:  joined = x r w u with r = 1 / sqrt(mean(x^2) + eps), u = act(gate);
// out = residual + s joined;  next = out r2 w2 with r2 = 1 / sqrt(mean(out^2) + eps).
// Backward, with D the gradient of out (that of next already added through the second norm):
//   second norm: dw2 += dn out r2,  D += r2 (a - out r2 mean(a out r2)) with a = dn w2;
//   dresidual = D;  ds += D joined;  dgate = D s x r w act'(gate);  dw += D s u x r;
//   dx = r (b - x r mean(b x r)) with b = D s u w.
// All of it is bound by memory: a row lives in the registers of its threads from the first load to the last store, so each
// tensor is read and written once and the sums over a row are exchanged by lane shuffles and, for rows of more than one wave,
// through a few floats of LDS.  32768 rows of 4096 channels in bf16 with gate, residual and second norm: forward 240 us, 5.6 TB/s,
// backward 440 us, 4.9 TB/s (a large copy: 5.1); 99900 rows of 56 in fp32: 13 and 25.
#include <algorithm>

#include "seq_common.hpp"

namespace psig {
namespace seq {
namespace {

struct NormArgs {
    const void *x, *gate, *residual, *weight, *scale, *next_weight;
    void *out, *next;
    float *stats;
    const void *grad_out, *grad_next;
    void *grad_x, *grad_gate, *grad_residual;
    float *partial;  // [3][blocks][C]: weight, scale, next_weight
    int64_t first_row, rows, x_stride, gate_stride, residual_stride;  // first_row: of a forward's launch
    int C, activation, float_params, want_weight, want_scale, want_next;
    float eps;
};

// Elements that a thread holds: EPT of them in vectors of E, the vectors of a row dealt to its TPR threads in turn, so that
// neighbouring threads read neighbouring vectors.
template <int TPR, int EPT, int E>
struct Deal {
    static constexpr int kVectors = EPT / E;
    static __device__ __forceinline__ int column(int v, int t) { return (v * TPR + t) * E; }
};

// a thread's share of a row as it lies in memory
template <typename T, int TPR, int EPT, int E>
struct RawRow {
    using D = Deal<TPR, EPT, E>;
    Pack<T, E> p[D::kVectors];
    __device__ __forceinline__ void load(const T *row, int t, int C) {
#pragma unroll
        for (int v = 0; v < D::kVectors; ++v) {
            const int c = D::column(v, t);
            p[v] = {};
            if (c < C) p[v] = *(const Pack<T, E> *)(row + c);  // (C is a multiple of E)
        }
    }
    __device__ __forceinline__ float at(int e) const { return to_float(p[e / E].v[e % E]); }
    __device__ __forceinline__ void get(float (&out)[EPT]) const {
#pragma unroll
        for (int v = 0; v < D::kVectors; ++v)
#pragma unroll
            for (int e = 0; e < E; ++e) out[v * E + e] = to_float(p[v].v[e]);
    }
};

template <typename T, int TPR, int EPT, int E>
__device__ __forceinline__ void load_row(float (&out)[EPT], const T *row, int t, int C) {
    RawRow<T, TPR, EPT, E> raw;
    raw.load(row, t, C);
    raw.get(out);
}

template <typename T, int TPR, int E>
__device__ __forceinline__ void store_vector(T *row, const float *x, int v, int t, int C) {
    const int c = (v * TPR + t) * E;
    if (c >= C) return;
    Pack<T, E> p;
#pragma unroll
    for (int e = 0; e < E; ++e) p.v[e] = from_float<T>(x[e]);
    *(Pack<T, E> *)(row + c) = p;
}

template <typename T, int TPR, int EPT, int E>
__device__ __forceinline__ void store_row(T *row, const float (&x)[EPT], int t, int C) {
#pragma unroll
    for (int v = 0; v < EPT / E; ++v) store_vector<T, TPR, E>(row, x + v * E, v, t, C);
}

// a parameter of the columns (NULL: `fill`), float32 or in the type of the rows
template <typename T, int TPR, int EPT, int E>
__device__ __forceinline__ void load_param(float (&out)[EPT], const void *p, int float_params, int t, int C, float fill) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < EPT; ++e) out[e] = fill;
    } else if (float_params) {
        load_row<float, TPR, EPT, E>(out, (const float *)p, t, C);
    } else {
        load_row<T, TPR, EPT, E>(out, (const T *)p, t, C);
    }
}

// Sum over the TPR threads of a row.  Where a row spans waves, through `slot` of LDS, which may be written again after a barrier;
// then every thread of the block has to come here.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float *slot) {
#pragma unroll
    for (int m = 1; m < (TPR < 64 ? TPR : 64); m <<= 1) x += __shfl_xor(x, m);
    if constexpr (TPR > 64) {
        constexpr int kWaves = TPR / 64;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x += slot[w];
    }
    return x;
}

// 1 / (1 + e^-g) and 1 minus it, which is not taken as a difference: behind g = 16 none of its digits would be left.  For rows in 32
// bits to a few units in the last place: the hardware's power of two, times 1 + r for what x = -g log2 e was rounded by.  For rows in
// bfloat16 without that, off by |g| units, 2^-17 at most where the answer is rounded to 2^-9.
struct Logistic {
    float up, down;
};
template <typename T>
__device__ __forceinline__ Logistic logistic(float g) {
    constexpr float kLog2e = 1.44269502162933349609375f, kLn2 = 0.693147182464599609375f, kLn2Rest = -1.904654299957767e-9f;
    const float x = -g * kLog2e;
    float t = __builtin_amdgcn_exp2f(x);
    if constexpr (sizeof(T) == 4) {
        const float r = fmaf(-x, kLn2Rest, fmaf(-x, kLn2, -g));
        t *= 1.f + __builtin_amdgcn_fmed3f(r, 0.f, r);  // (zero instead of NaN where g is infinite)
    }
    const float up = __builtin_amdgcn_rcpf(1.f + t);
    return {up, fminf(t, 1e38f) * up};  // (where t is infinite `up` is zero, and so is all that either is used for)
}

template <typename T>
__device__ __forceinline__ float gate_value(float g, int activation) {
    if (activation == PATHSIG_GATE_LINEAR) return g;
    const float s = logistic<T>(g).up;
    return activation == PATHSIG_GATE_SILU ? g * s : s;
}

// value and derivative
template <typename T>
__device__ __forceinline__ void gate_both(float g, int activation, float &u, float &du) {
    if (activation == PATHSIG_GATE_LINEAR) {
        u = g;
        du = 1.f;
        return;
    }
    const Logistic s = logistic<T>(g);
    if (activation == PATHSIG_GATE_SILU) {
        u = g * s.up;
        du = s.up + u * s.down;
    } else {
        u = s.up;
        du = s.up * s.down;
    }
}

// rows of up to a wave's threads share a block of four waves, wider ones have one to themselves
constexpr int threads_of(int threads_per_row) { return threads_per_row <= 64 ? 256 : threads_per_row; }

template <typename T, int TPR, int EPT, int E>
__global__ __launch_bounds__(threads_of(TPR)) void norm_forward_kernel(const NormArgs a) {
    constexpr int kRows = threads_of(TPR) / TPR;
    __shared__ float slots[2][16];
    const int t = threadIdx.x % TPR;
    const int64_t row_or_behind = a.first_row + (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool live = row_or_behind < a.rows;  // (all threads of a block meet at barriers)
    const int64_t row = live ? row_or_behind : a.rows - 1;
    const int C = a.C;
    float x[EPT], w[EPT];
    load_row<T, TPR, EPT, E>(x, (const T *)a.x + row * a.x_stride, t, C);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) sum += x[e] * x[e];
    const float r = 1.f / sqrtf(row_sum<TPR>(sum, slots[0]) / (float)C + a.eps);
    load_param<T, TPR, EPT, E>(w, a.weight, a.float_params, t, C, 1.f);
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = x[e] * r * w[e];
    if (a.gate) {
        load_row<T, TPR, EPT, E>(w, (const T *)a.gate + row * a.gate_stride, t, C);
#pragma unroll
        for (int e = 0; e < EPT; ++e) x[e] *= gate_value<T>(w[e], a.activation);
    }
    if (a.scale) {
        load_param<T, TPR, EPT, E>(w, a.scale, a.float_params, t, C, 1.f);
#pragma unroll
        for (int e = 0; e < EPT; ++e) x[e] *= w[e];
    }
    if (a.residual) {
        load_row<T, TPR, EPT, E>(w, (const T *)a.residual + row * a.residual_stride, t, C);
#pragma unroll
        for (int e = 0; e < EPT; ++e) x[e] += w[e];
    }
    if (live) store_row<T, TPR, EPT, E>((T *)a.out + row * C, x, t, C);
    if (live && a.stats && t == 0) a.stats[row] = r;
    if (!a.next) return;
    // (columns behind the last hold zeros: they were loaded as zeros, and gates and scales only multiply)
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) sum += x[e] * x[e];
    const float r2 = 1.f / sqrtf(row_sum<TPR>(sum, slots[1]) / (float)C + a.eps);
    load_param<T, TPR, EPT, E>(w, a.next_weight, a.float_params, t, C, 1.f);
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = x[e] * r2 * w[e];
    if (!live) return;
    store_row<T, TPR, EPT, E>((T *)a.next + row * C, x, t, C);
    if (a.stats && t == 0) a.stats[a.rows + row] = r2;
}

// Waves to a SIMD that the backward is compiled for and launched with: what its registers allow without spilling.  Rows that have a
// block to themselves have their addresses in scalar registers.
constexpr int backward_waves(int element, int threads_per_row) {
    if (threads_per_row > 256) return 4;
    return element == 4 && threads_per_row <= 64 ? 2 : 3;
}

// Blocks take rows in turn and hold the sums over their rows of the parameters' gradients in registers; norm_columns_kernel
// adds the blocks in a fixed order (6 to 7 us at 32768 rows of 2048 and 4096).
template <typename T, int TPR, int EPT, int E>
__global__ __launch_bounds__(TPR > 256 ? 1024 : threads_of(TPR), backward_waves(sizeof(T), TPR)) void norm_backward_kernel(const NormArgs a) {
    constexpr int kRows = threads_of(TPR) / TPR;
    using D = Deal<TPR, EPT, E>;
    __shared__ float slots[2][16];
    const int t = kRows > 1 ? threadIdx.x % TPR : threadIdx.x;
    const int C = a.C;
    float sum_w[EPT] = {}, sum_s[EPT] = {}, sum_n[EPT] = {};
    // The tensors of a row are loaded while the row before is worked on; not those of wide rows in 32 bits, for which the 128 registers
    // of a thread there are too few (8192 x 4096: with 100 to 120 bytes of them spilled 406 to 514 us a step, without 333).
    constexpr bool kAhead = !(sizeof(T) == 4 && TPR > 256);
    RawRow<T, TPR, EPT, E> raw_x, raw_d, raw_u, raw_out, raw_n;
    float raw_r = 0.f, raw_r2 = 0.f;
    // (a row behind the last is one of zeros, which adds nothing)
    auto fetch = [&](int64_t row) {
        const bool live = row < a.rows;
        const int have = live ? C : 0;
        raw_x.load((const T *)a.x + row * a.x_stride, t, have);
        raw_r = live ? a.stats[row] : 0.f;
        if (a.grad_out) raw_d.load((const T *)a.grad_out + row * C, t, have);
        if (a.gate) raw_u.load((const T *)a.gate + row * a.gate_stride, t, have);
        if (a.grad_next) {
            if (a.residual) raw_out.load((const T *)a.residual + row * a.residual_stride, t, have);
            raw_n.load((const T *)a.grad_next + row * C, t, have);
            raw_r2 = live ? a.stats[a.rows + row] : 0.f;
        }
    };
    const int64_t step = (int64_t)gridDim.x * kRows;
    const int own = kRows > 1 ? threadIdx.x / TPR : 0;
    if (kAhead) fetch((int64_t)blockIdx.x * kRows + own);
    // as many turns for every thread of a block: they meet at barriers
    for (int64_t first = (int64_t)blockIdx.x * kRows; first < a.rows; first += step) {
        const int64_t row = first + own;
        const bool live = row < a.rows;
        if (!kAhead) fetch(row);
        RawRow<T, TPR, EPT, E> x = raw_x, d = raw_d, u = raw_u, residual = raw_out, n = raw_n;
        const float r = raw_r, r2 = raw_r2;
        if (kAhead && first + step < a.rows) fetch(row + step);
        // (read again for every row, from the cache: held, the parameters would take 24 registers)
        const void *weight = a.weight, *scale = a.scale, *next_weight = a.next_weight;
        asm volatile("" : "+s"(weight), "+s"(scale), "+s"(next_weight));
        float unit[EPT], w[EPT], p[EPT], up[EPT];
        load_param<T, TPR, EPT, E>(w, weight, a.float_params, t, C, 1.f);
        load_param<T, TPR, EPT, E>(p, scale, a.float_params, t, C, 1.f);
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
            unit[e] = x.at(e) * r;
            up[e] = a.grad_out ? d.at(e) : 0.f;
        }
        if (a.grad_next) {
            // out as the forward had it before rounding, from the same inputs
            float unit2[EPT], dn[EPT], nw[EPT];
            load_param<T, TPR, EPT, E>(nw, next_weight, a.float_params, t, C, 1.f);
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const float g = a.gate ? gate_value<T>(u.at(e), a.activation) : 1.f;
                unit2[e] = ((a.residual ? residual.at(e) : 0.f) + unit[e] * w[e] * g * p[e]) * r2;
                dn[e] = n.at(e);
                sum_n[e] += dn[e] * unit2[e];
                dn[e] *= nw[e];
                dot += dn[e] * unit2[e];
            }
            dot = row_sum<TPR>(dot, slots[0]) / (float)C;
#pragma unroll
            for (int e = 0; e < EPT; ++e) up[e] += r2 * (dn[e] - unit2[e] * dot);
        }
        if (live && a.grad_residual) store_row<T, TPR, EPT, E>((T *)a.grad_residual + row * C, up, t, C);
        if (a.gate) {
            float to_gate[EPT];
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                float g, dg;
                gate_both<T>(u.at(e), a.activation, g, dg);
                const float normed = unit[e] * w[e];
                sum_s[e] += up[e] * normed * g;
                up[e] *= p[e];
                to_gate[e] = up[e] * normed * dg;
                up[e] *= g;
            }
            if (live && a.grad_gate) store_row<T, TPR, EPT, E>((T *)a.grad_gate + row * C, to_gate, t, C);
        } else {
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                sum_s[e] += up[e] * unit[e] * w[e];
                up[e] *= p[e];
            }
        }
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
            sum_w[e] += up[e] * unit[e];
            up[e] *= w[e];
            dot += up[e] * unit[e];
        }
        // (the other slot than above: a wave that is ahead may write it while others still read the first)
        dot = row_sum<TPR>(dot, slots[1]) / (float)C;
#pragma unroll
        for (int e = 0; e < EPT; ++e) up[e] = r * (up[e] - unit[e] * dot);
        if (live && a.grad_x) store_row<T, TPR, EPT, E>((T *)a.grad_x + row * C, up, t, C);
        if (TPR > 64) __syncthreads();  // before slots are written again
    }
    if (!a.partial) return;
    const int64_t plane = (int64_t)gridDim.x * C;
    float *mine = a.partial + (int64_t)blockIdx.x * C;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int v = 0; v < D::kVectors; ++v)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = D::column(v, t) + e;
                if (c >= C) continue;
                if (a.want_weight) mine[c] = sum_w[v * E + e];
                if (a.want_scale) mine[plane + c] = sum_s[v * E + e];
                if (a.want_next) mine[2 * plane + c] = sum_n[v * E + e];
            }
    } else {
        // the rows of a block meet in LDS, one parameter after the other
        __shared__ float meet[kRows][TPR * EPT];
        const int which = threadIdx.x / TPR;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (!(k == 0 ? a.want_weight : k == 1 ? a.want_scale : a.want_next)) continue;
            __syncthreads();
#pragma unroll
            for (int v = 0; v < D::kVectors; ++v)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    meet[which][D::column(v, t) + e] = (k == 0 ? sum_w : k == 1 ? sum_s : sum_n)[v * E + e];
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += 256) {
                float s = 0.f;
#pragma unroll 4
                for (int i = 0; i < kRows; ++i) s += meet[i][c];
                mine[k * plane + c] = s;
            }
        }
    }
}

constexpr int kColumnLanes = 32, kColumnParts = 8;

template <typename P>
__global__ __launch_bounds__(kColumnLanes * kColumnParts) void norm_columns_kernel(const float *partial, int64_t blocks, int C,
                                                                                  P *weight, P *scale, P *next_weight) {
    __shared__ float meet[kColumnParts][kColumnLanes];
    P *const out = blockIdx.y == 0 ? weight : blockIdx.y == 1 ? scale : next_weight;
    if (!out) return;
    const int c = blockIdx.x * kColumnLanes + threadIdx.x, part = threadIdx.y;
    float s = 0.f;
    if (c < C) {
        const float *p = partial + blockIdx.y * blocks * C + c;
#pragma unroll 4
        for (int64_t i = part; i < blocks; i += kColumnParts) s += p[i * C];
    }
    meet[part][threadIdx.x] = s;
    __syncthreads();
    if (part > 0 || c >= C) return;
#pragma unroll
    for (int i = 1; i < kColumnParts; ++i) s += meet[i][threadIdx.x];
    out[c] = from_float<P>(s);
}

// Elements that a thread holds, of rows of up to 8192 channels.
constexpr int kElements = 8;

// The fewest threads that hold a row.
int threads_per_row(int64_t C) {
    int threads = 8;
    while (threads < 1024 && (int64_t)threads * kElements < C) threads *= 2;
    return threads;
}

int rows_per_block(int threads) { return threads_of(threads) / threads; }

// Blocks of the backward: as many as the device holds at once, and the rows dealt evenly to them.
int64_t backward_blocks(int dtype, int64_t rows, int64_t C) {
    const int per_row = threads_per_row(C), threads = threads_of(per_row);
    const int64_t groups = ceil_div(rows, rows_per_block(per_row));
    const int waves = backward_waves(dtype == PATHSIG_F32 ? 4 : 2, per_row);
    const int64_t most = (int64_t)256 * (256 * waves / threads);
    return ceil_div(groups, ceil_div(groups, most));
}

template <typename T, int TPR, int E>
void launch(const NormArgs &a, bool backward, int64_t blocks, hipStream_t stream) {
    constexpr int kThreads = threads_of(TPR);
    if (backward)
        norm_backward_kernel<T, TPR, kElements, E><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a);
    else
        norm_forward_kernel<T, TPR, kElements, E><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a);
}

template <typename T, int E>
void dispatch(const NormArgs &a, bool backward, int64_t blocks, hipStream_t stream) {
    switch (threads_per_row(a.C)) {
        case 8: return launch<T, 8, E>(a, backward, blocks, stream);
        case 16: return launch<T, 16, E>(a, backward, blocks, stream);
        case 32: return launch<T, 32, E>(a, backward, blocks, stream);
        case 64: return launch<T, 64, E>(a, backward, blocks, stream);
        case 128: return launch<T, 128, E>(a, backward, blocks, stream);
        case 256: return launch<T, 256, E>(a, backward, blocks, stream);
        case 512: return launch<T, 512, E>(a, backward, blocks, stream);
        default: return launch<T, 1024, E>(a, backward, blocks, stream);
    }
}

int check_norm(const pathsig_norm *c) {
    if (!c) {
        set_error("call must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->dtype != PATHSIG_F32 && c->dtype != PATHSIG_BF16) {
        set_error("dtype must be PATHSIG_F32 or PATHSIG_BF16");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->param_dtype != PATHSIG_F32 && c->param_dtype != c->dtype) {
        set_error("param_dtype must be PATHSIG_F32 or the dtype of the rows");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->activation < PATHSIG_GATE_SILU || c->activation > PATHSIG_GATE_LINEAR) {
        set_error("unknown activation %d", c->activation);
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->rows < 0 || c->C < 1) {
        set_error("rows must be >= 0 and C >= 1 (got %lld, %lld)", (long long)c->rows, (long long)c->C);
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->x_stride < 0 || c->gate_stride < 0 || c->residual_stride < 0) {
        set_error("row strides must not be negative");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (!(c->eps >= 0.f)) {
        set_error("eps must not be negative");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->C > PATHSIG_MAX_NORM_CHANNELS) {
        set_error("C must be at most %d (got %lld)", PATHSIG_MAX_NORM_CHANNELS, (long long)c->C);
        return PATHSIG_ERR_UNSUPPORTED;
    }
    if (ceil_div(c->rows, rows_per_block(threads_per_row(c->C))) > 0x7fffffff) {
        set_error("too many rows (%lld)", (long long)c->rows);
        return PATHSIG_ERR_UNSUPPORTED;
    }
    return PATHSIG_OK;
}

NormArgs norm_args(const pathsig_norm *c) {
    NormArgs a = {};
    a.x = c->x;
    a.gate = c->gate;
    a.residual = c->residual;
    a.weight = c->weight;
    a.scale = c->scale;
    a.next_weight = c->next_weight;
    a.rows = c->rows;
    a.C = (int)c->C;
    a.x_stride = c->x_stride;
    a.gate_stride = c->gate_stride;
    a.residual_stride = c->residual_stride;
    a.activation = c->activation;
    a.float_params = c->param_dtype == PATHSIG_F32;
    a.eps = c->eps;
    return a;
}

// Vectors of 16 bytes where every row of every tensor starts at a multiple of 16 bytes (parameters too, whose vectors of E
// elements are as wide or wider); else single elements, which any address allows.
bool vectors(const NormArgs &a, int element) {
    const int64_t E = 16 / element;
    const void *const all[] = {a.x, a.gate, a.residual, a.weight, a.scale, a.next_weight, a.out, a.next,
                               a.grad_out, a.grad_next, a.grad_x, a.grad_gate, a.grad_residual};
    for (const void *p : all)
        if (!aligned16(p)) return false;
    return a.C % E == 0 && a.x_stride % E == 0 && a.gate_stride % E == 0 && a.residual_stride % E == 0;
}

void run(const NormArgs &a, int dtype, bool backward, int64_t blocks, hipStream_t stream) {
    if (dtype == PATHSIG_F32) {
        if (vectors(a, 4)) return dispatch<float, 4>(a, backward, blocks, stream);
        return dispatch<float, 1>(a, backward, blocks, stream);
    }
    if (vectors(a, 2)) return dispatch<bf16, 8>(a, backward, blocks, stream);
    return dispatch<bf16, 1>(a, backward, blocks, stream);
}

}  // namespace
}  // namespace seq
}  // namespace psig

using namespace psig;
using namespace psig::seq;

extern "C" {

int pathsig_norm_forward(const pathsig_norm *call, void *out, void *next, float *statistics, void *stream) {
    if (const int rc = check_norm(call)) return rc;
    if (call->rows == 0) return PATHSIG_OK;
    if (!call->x || !out) {
        set_error("x and out must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    NormArgs a = norm_args(call);
    a.out = out;
    a.next = next;
    a.stats = statistics;
    // (a launch has fewer than 2^32 threads)
    const int64_t of_block = rows_per_block(threads_per_row(a.C)), most = ((int64_t)1 << 31) / threads_of(threads_per_row(a.C));
    for (; a.first_row < a.rows; a.first_row += most * of_block)
        run(a, call->dtype, false, std::min(ceil_div(a.rows - a.first_row, of_block), most), (hipStream_t)stream);
    return launch_status("norm forward");
}

size_t pathsig_norm_backward_workspace(const pathsig_norm *call) {
    if (check_norm(call) != PATHSIG_OK || call->rows == 0) return 0;
    return (size_t)3 * backward_blocks(call->dtype, call->rows, call->C) * call->C * sizeof(float);
}

int pathsig_norm_backward(const pathsig_norm *call, const float *statistics, const void *grad_out, const void *grad_next,
                          void *grad_x, void *grad_gate, void *grad_residual, void *grad_weight, void *grad_scale,
                          void *grad_next_weight, void *workspace, size_t workspace_bytes, void *stream) {
    if (const int rc = check_norm(call)) return rc;
    const bool params = grad_weight || grad_scale || grad_next_weight;
    if (call->rows > 0 && (!call->x || !statistics)) {
        set_error("x and statistics must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (grad_gate && !call->gate) {
        set_error("grad_gate is asked for, but there is no gate");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (params && call->rows > 0 && (!workspace || workspace_bytes < pathsig_norm_backward_workspace(call))) {
        set_error("norm backward: workspace of %zu bytes needed, got %zu", pathsig_norm_backward_workspace(call),
                  workspace ? workspace_bytes : (size_t)0);
        return PATHSIG_ERR_WORKSPACE;
    }
    NormArgs a = norm_args(call);
    const int64_t blocks = call->rows > 0 ? backward_blocks(call->dtype, a.rows, a.C) : 0;
    if (call->rows > 0) {
        a.stats = const_cast<float *>(statistics);
        a.grad_out = grad_out;
        a.grad_next = grad_next;
        a.grad_x = grad_x;
        a.grad_gate = grad_gate;
        a.grad_residual = grad_residual;
        a.partial = params ? (float *)workspace : nullptr;
        a.want_weight = grad_weight != nullptr;
        a.want_scale = grad_scale != nullptr;
        a.want_next = grad_next_weight != nullptr;
        run(a, call->dtype, true, blocks, (hipStream_t)stream);
        if (const int rc = launch_status("norm backward")) return rc;
    }
    if (!params) return PATHSIG_OK;
    const dim3 grid((unsigned)ceil_div(a.C, kColumnLanes), 3), block(kColumnLanes, kColumnParts);
    if (call->param_dtype == PATHSIG_F32)
        norm_columns_kernel<float><<<grid, block, 0, (hipStream_t)stream>>>((const float *)workspace, blocks, a.C, (float *)grad_weight,
                                                                          (float *)grad_scale, (float *)grad_next_weight);
    else
        norm_columns_kernel<bf16><<<grid, block, 0, (hipStream_t)stream>>>((const float *)workspace, blocks, a.C, (bf16 *)grad_weight,
                                                                         (bf16 *)grad_scale, (bf16 *)grad_next_weight);
    return launch_status("norm backward, parameters");
}

}  // extern "C"
