// Linear attention with a decay for each head: whole sequences, their gradients, and single tokens (pathsig_linattn_* of
// pathsig_hip.h).
//
// Recurrence of a head, state S [Dk, Dv]:  S_t = e^g S_(t-1) + k_t v_t^T,  o_t = scale S_t^T q_t.
// Gradients, with R_t = dL/dS_t through the outputs from t on:  R_t = e^g R_(t+1) + scale q_t do_t^T,
//   dq_t = scale S_t do_t,   dk_t = R_t v_t,   dv_t = R_t^T k_t,   dS_(-1) = e^g R_0,
//   dg = sum over t of e^g <S_(t-1), R_t>, worked out inside chunks and pieces as seq_chunks.hip says.
// So all three gradients are the forward's recurrence with other tensors in the places of q, k and v: dq with (do, v, k),
// dv backwards in time with (k, q, do), dk backwards in time with (v, do, q).
//
// A sweep over whole sequences is cut into pieces where there are fewer heads of sequences than the device takes at once: the
// states that the pieces add from zero (k and v read once more), a scan over the pieces, and all pieces at once from their
// states.
#include <algorithm>

#include "seq_attention.hpp"

namespace psig {
namespace seq {
namespace {

// starts[s] holds what piece s - 1 adds; in place becomes the state in front of piece s.  Vectors of V elements with a thread each:
// bound by reading and writing `starts`, a thread's chain of pieces one after the other (65536 tokens, 8 heads of 128 x 128: 20 us).
template <int V>
__global__ __launch_bounds__(256) void join_kernel(const Sweep a) {
    using P = Pack<float, V>;
    const int64_t plane = (int64_t)a.Dk * a.Dv;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (i >= plane) return;
    const int h = blockIdx.y;
    const int64_t b = blockIdx.z, head = (b * a.H + h) * plane, stride = a.B * a.H * plane;
    const int64_t n = length_of(a.lengths, b, a.L);
    const float g2 = decay_of(a.log_decay, h) * kLog2e;
    float *const p = a.starts + head + i;
    P x = {};
    if (a.first) {
#pragma unroll
        for (int e = 0; e < V; ++e) x.v[e] = a.first[head + i + e];
    }
    *(P *)p = x;
    constexpr int kBatch = 16;  // loads on their way at once (stores of one and loads of the next may meet, for all the compiler knows)
    for (int s0 = 1; s0 < a.pieces; s0 += kBatch) {
        P add[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (s0 + j < a.pieces) add[j] = *(const P *)(p + (s0 + j) * stride);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (s0 + j >= a.pieces) break;
            const Range before = range_of(a, n, s0 + j - 1);
            // (nothing of the zeros in front of the first token, whatever the decay)
            const float f = s0 + j == 1 && !a.first ? 0.f : exp2f(g2 * (float)(before.end - before.begin));
#pragma unroll
            for (int e = 0; e < V; ++e) x.v[e] = x.v[e] * f + add[j].v[e];
            *(P *)(p + (s0 + j) * stride) = x;
        }
    }
}

// The state in front of the first token, for a call that writes the last state over it: with few pieces every block of a sweep reads
// the first one, in no order with the block that writes the last.
__global__ void copy_state_kernel(const float *from, float *to, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from[i];
}

// The parts of a head's gradient, in a fixed order and in 64 bits; a few thousand numbers at most, bound by the launch.
__global__ void decay_sum_kernel(const float *partial, int64_t rows, int H, float *out) {
    const int h = blockIdx.x;
    double s = 0;
    for (int64_t i = threadIdx.x; i < rows; i += 64) s += partial[i * H + h];
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m);
    if (threadIdx.x == 0) out[h] = (float)s;
}

// [rows, H, D] float -> [rows, H / group, D]: the gradient of a key is the sum over the heads that read it, in their order (no
// atomics).  Bound by reading `in` (50 x 333 tokens, 6 heads of 40 and 56, 3 of keys, fp32: 7 us each).
template <typename T>
__global__ void group_sum_kernel(const float *in, T *out, int64_t rows, int Hkv, int group, int D) {
    const int64_t n = rows * Hkv * D;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t head = i / D;
        const float *p = in + head * group * D + i % D;
        float s = 0.f;
        for (int g = 0; g < group; ++g) s += p[(int64_t)g * D];
        out[i] = from_float<T>(s);
    }
}

// One token.  A block has a head of a sequence: TX threads along Dv, the rows of the state dealt to the 256 / TX groups of
// threads, so that the state is read and written once, in lines.  Bound by that: 128 sequences, 16 heads of 128 x 128 take 60 us,
// 4.5 TB/s; a single sequence is bound by the launch (5 us a call).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void step_kernel(const Sweep a, float *state, int tx_log2) {
    __shared__ float qs[PATHSIG_MAX_HEAD_DIM], ks[PATHSIG_MAX_HEAD_DIM];
    __shared__ float meet[256 * VEC];
    using V = Pack<float, VEC>;
    const int h = blockIdx.x, tid = threadIdx.x;
    const int64_t b = blockIdx.y;
    const T *q = (const T *)a.q.p + b * a.q.sb + (h / a.q.group) * a.q.sh;
    const T *k = (const T *)a.k.p + b * a.k.sb + (h / a.k.group) * a.k.sh;
    const T *v = (const T *)a.v.p + b * a.v.sb + (h / a.v.group) * a.v.sh;
    if (tid < a.Dk) {
        qs[tid] = to_float(q[tid]) * a.out_scale;
        ks[tid] = to_float(k[tid]);
    }
    __syncthreads();
    const float decay = expf(decay_of(a.log_decay, h));
    const int TX = 1 << tx_log2, TY = 256 >> tx_log2;
    const int tx = tid & (TX - 1), ty = tid >> tx_log2;
    float *S = state + (b * a.H + h) * a.Dk * a.Dv;
    T *out = (T *)a.out + (b * a.H + h) * a.Dv;
    for (int c0 = 0; c0 < a.Dv; c0 += TX * VEC) {
        const int c = c0 + tx * VEC;
        const bool mine = c < a.Dv;
        float vc[VEC], o[VEC] = {};
#pragma unroll
        for (int e = 0; e < VEC; ++e) vc[e] = mine ? to_float(v[c + e]) : 0.f;
        if (mine) {
#pragma unroll 8
            for (int r = ty; r < a.Dk; r += TY) {
                V s = *(const V *)(S + (int64_t)r * a.Dv + c);
                const float kr = ks[r], qr = qs[r];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    s.v[e] = s.v[e] * decay + kr * vc[e];
                    o[e] += qr * s.v[e];
                }
                *(V *)(S + (int64_t)r * a.Dv + c) = s;
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) meet[tid * VEC + e] = o[e];
        __syncthreads();
        for (int i = tid; i < TX * VEC; i += 256) {
            if (c0 + i >= a.Dv) continue;
            float s = 0.f;
            for (int y = 0; y < TY; ++y) s += meet[y * TX * VEC + i];
            out[c0 + i] = from_float<T>(s);
        }
        __syncthreads();
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------
int check_call(const pathsig_linattn *c) {
    if (!c) {
        set_error("call must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->dtype != PATHSIG_F32 && c->dtype != PATHSIG_BF16) {
        set_error("dtype must be PATHSIG_F32 or PATHSIG_BF16");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->B < 0 || c->L < 0 || c->H < 1 || c->Hkv < 1 || c->H % c->Hkv) {
        set_error("sizes must not be negative and H a multiple of Hkv (got B %lld, L %lld, H %lld, Hkv %lld)", (long long)c->B,
                  (long long)c->L, (long long)c->H, (long long)c->Hkv);
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->Dk < 1 || c->Dv < 1) {
        set_error("Dk and Dv must be at least 1 (got %lld, %lld)", (long long)c->Dk, (long long)c->Dv);
        return PATHSIG_ERR_ARGUMENT;
    }
    if (c->Dk > PATHSIG_MAX_HEAD_DIM || c->Dv > PATHSIG_MAX_HEAD_DIM) {
        set_error("Dk and Dv must be at most %d (got %lld, %lld)", PATHSIG_MAX_HEAD_DIM, (long long)c->Dk, (long long)c->Dv);
        return PATHSIG_ERR_UNSUPPORTED;
    }
    if (c->H > 65535 || c->B > 65535 || c->L > 0x7fffffff) {
        set_error("at most 65535 sequences and heads and 2^31 - 1 tokens (got B %lld, H %lld, L %lld)", (long long)c->B,
                  (long long)c->H, (long long)c->L);
        return PATHSIG_ERR_UNSUPPORTED;
    }
    if (std::max({c->q_stride[1], c->k_stride[1], c->v_stride[1]}) > PATHSIG_MAX_TOKEN_STRIDE || c->H * std::max(c->Dk, c->Dv) > PATHSIG_MAX_TOKEN_STRIDE) {
        set_error("tokens may be at most %d elements apart", PATHSIG_MAX_TOKEN_STRIDE);
        return PATHSIG_ERR_UNSUPPORTED;
    }
    for (int i = 0; i < 3; ++i)
        if (c->q_stride[i] < 0 || c->k_stride[i] < 0 || c->v_stride[i] < 0) {
            set_error("strides must not be negative");
            return PATHSIG_ERR_ARGUMENT;
        }
    if (!c->log_decay) {
        set_error("log_decay must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    return PATHSIG_OK;
}

View view(const void *p, const int64_t *stride, int64_t group) { return {p, stride[0], stride[1], stride[2], (int)group}; }

View dense(const void *p, int64_t L, int64_t heads, int64_t D, int64_t group) {
    return {p, L * heads * D, heads * D, D, (int)group};
}

int64_t element_of(const pathsig_linattn *c) { return c->dtype == PATHSIG_F32 ? 4 : 2; }
// channels in whole units of 16 bytes
int64_t padded(const pathsig_linattn *c, int64_t D) { return ceil_div(D * element_of(c), 16) * 16 / element_of(c); }

// q, k and v do not lie in whole units of 16 bytes
bool copied(const pathsig_linattn *c) {
    const int64_t E = 16 / element_of(c);
    int64_t odd = c->Dk % E + c->Dv % E;
    for (int i = 0; i < 3; ++i) odd += c->q_stride[i] % E + c->k_stride[i] % E + c->v_stride[i] % E;
    return odd > 0;
}

// Pieces of a call's sweeps, the same for all of them: as many as bring two waves to each of the 1024 SIMDs (a block has a wave for
// 32 columns of the state, up to four; four waves in fp32: 50 x 333, 6 heads of 40 x 56, 353 -> 393 us a step), of whole chunks, and not so short that what a piece costs (its state written and read,
// 8 Dk Dv bytes) is more than what its tokens do.  Two pieces of blocks of four waves are folded in halves, or every second compute
// unit would have no block to fold with.
void cut(const pathsig_linattn *c, int64_t *piece, int *pieces, int *run) {
    const int64_t wide = std::max(c->Dk, c->Dv), waves = wide <= 32 ? 1 : wide <= 64 ? 2 : 4;
    const int64_t blocks = std::max<int64_t>(c->B * c->H, 1), element = element_of(c);
    const int64_t least = std::max<int64_t>(64, 8 * c->Dk * c->Dv / (element * (c->Dk + c->Dv)));
    const int64_t want = std::max<int64_t>(1, std::min(2048 / waves / blocks, c->L / least));
    *run = want == 2 && waves == 4 && c->L >= 4 * least ? 2 : 1;
    const int64_t count = want * *run;
    *piece = std::max<int64_t>(ceil_div(ceil_div(c->L, count), 64) * 64, 64);
    *pieces = (int)(*run * std::max<int64_t>(ceil_div(c->L, *piece * *run), 1));
}

size_t starts_bytes(const pathsig_linattn *c) {
    int64_t piece;
    int pieces, run;
    cut(c, &piece, &pieces, &run);
    return pieces > 1 ? (size_t)pieces * c->B * c->H * c->Dk * c->Dv * sizeof(float) : 0;
}

Sweep sweep_of(const pathsig_linattn *c) {
    Sweep a = {};
    a.log_decay = c->log_decay;
    a.lengths = c->lengths;
    a.B = c->B;
    a.L = c->L;
    a.H = (int)c->H;
    a.Dk = (int)c->Dk;
    a.Dv = (int)c->Dv;
    a.Kp = (int)padded(c, c->Dk);
    a.Vp = (int)padded(c, c->Dv);
    a.in_scale = 1.f;
    a.out_scale = 1.f;
    a.row = c->Dv;
    a.column = 1;
    cut(c, &a.piece, &a.pieces, &a.run);
    return a;
}

template <typename T>
void chunks(const Sweep &a, bool fold, hipStream_t stream) {
    if (a.Dk <= 32) return launch_chunks<T, 1>(a, fold, stream);
    if (a.Dk <= 64) return launch_chunks<T, 2>(a, fold, stream);
    if (a.Dk <= 128) return launch_chunks<T, 4>(a, fold, stream);
    launch_chunks<T, 8>(a, fold, stream);
}

// the states in front of the pieces
template <typename T>
void fold(Sweep &a, float *starts, hipStream_t stream) {
    a.starts = starts;
    if (a.pieces == 1) return;
    chunks<T>(a, true, stream);
    if (a.pieces <= kJoinInside) return;
    const int64_t plane = (int64_t)a.Dk * a.Dv;
    if (plane % 4 == 0)
        join_kernel<4><<<dim3((unsigned)ceil_div(plane, 1024), a.H, (unsigned)a.B), 256, 0, stream>>>(a);
    else
        join_kernel<1><<<dim3((unsigned)ceil_div(plane, 256), a.H, (unsigned)a.B), 256, 0, stream>>>(a);
}

template <typename T>
void decay(const Sweep &a, const Sweep &back, const View &grad_out, float *partial, hipStream_t stream) {
    if (a.Dk <= 32) return launch_decay<T, 1>(a, back, grad_out, partial, stream);
    if (a.Dk <= 64) return launch_decay<T, 2>(a, back, grad_out, partial, stream);
    launch_decay<T, 4>(a, back, grad_out, partial, stream);
}

size_t place(size_t &total, size_t bytes) {
    const size_t at = total;
    total += (bytes + 255) / 256 * 256;
    return at;
}

// what a forward's workspace holds: the states in front of the pieces, and q, k and v where they are copied
struct ForwardLayout {
    size_t starts, q, k, v, total;  // byte offsets
};

ForwardLayout forward_layout(const pathsig_linattn *c) {
    ForwardLayout l = {};
    l.starts = place(l.total, starts_bytes(c));
    if (copied(c)) {
        const size_t tokens = (size_t)c->B * c->L * element_of(c), K = padded(c, c->Dk), V = padded(c, c->Dv);
        l.q = place(l.total, tokens * c->H * K);
        l.k = place(l.total, tokens * c->Hkv * K);
        l.v = place(l.total, tokens * c->Hkv * V);
    }
    return l;
}

struct Copy {
    const void *from;
    void *to;
    int64_t sb, st, sh;
    int heads, D, padded;
};
struct Copies {
    Copy c[3];
};

// Rows of D channels to rows of whole units, the rest zeros; a thread has a unit.  Tokens behind the end of a sequence are left out.
template <typename T>
__global__ __launch_bounds__(256) void copy_kernel(const Copies copies, int64_t L, const int32_t *lengths) {
    constexpr int E = 16 / (int)sizeof(T);
    const Copy &c = copies.c[blockIdx.z];
    const int64_t b = blockIdx.y, n = length_of(lengths, b, L), per_token = (int64_t)c.heads * (c.padded / E);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n * per_token; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per_token, in_token = i % per_token;
        const int h = (int)(in_token / (c.padded / E)), at = (int)(in_token % (c.padded / E)) * E;
        const T *const from = (const T *)c.from + b * c.sb + t * c.st + h * c.sh + at;
        Pack<T, E> unit = {};
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (at + e < c.D) unit.v[e] = from[e];
        *(Pack<T, E> *)((T *)c.to + ((b * L + t) * c.heads + h) * c.padded + at) = unit;
    }
}

template <typename T>
void copy(const pathsig_linattn *c, const Copy *list, int count, hipStream_t stream) {
    if (c->L == 0) return;
    Copies all = {};
    int64_t most = 0;
    for (int i = 0; i < count; ++i) {
        all.c[i] = list[i];
        most = std::max(most, c->L * list[i].heads * list[i].padded * (int64_t)sizeof(T) / 16);
    }
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(most, 256), std::max<int64_t>(1, 4096 / c->B));
    copy_kernel<T><<<dim3(blocks, (unsigned)c->B, (unsigned)count), 256, 0, stream>>>(all, c->L, c->lengths);
}

struct Inputs {
    View q, k, v;
};

// q, k and v as the sweeps read them: in place, or copied into (or already in) a forward's workspace
template <typename T>
Inputs inputs(const pathsig_linattn *c, const void *q, const void *k, const void *v, char *ws, bool there, hipStream_t stream) {
    const int64_t group = c->H / c->Hkv;
    if (!copied(c)) return {view(q, c->q_stride, 1), view(k, c->k_stride, group), view(v, c->v_stride, group)};
    const ForwardLayout l = forward_layout(c);
    const int64_t K = padded(c, c->Dk), V = padded(c, c->Dv);
    if (!there) {
        const int H = (int)c->H, Hkv = (int)c->Hkv, Dk = (int)c->Dk, Dv = (int)c->Dv;
        const Copy list[3] = {{q, ws + l.q, c->q_stride[0], c->q_stride[1], c->q_stride[2], H, Dk, (int)K},
                              {k, ws + l.k, c->k_stride[0], c->k_stride[1], c->k_stride[2], Hkv, Dk, (int)K},
                              {v, ws + l.v, c->v_stride[0], c->v_stride[1], c->v_stride[2], Hkv, Dv, (int)V}};
        copy<T>(c, list, 3, stream);
    }
    return {dense(ws + l.q, c->L, c->H, K, 1), dense(ws + l.k, c->L, c->Hkv, K, group), dense(ws + l.v, c->L, c->Hkv, V, group)};
}

// pointers that are read in whole units where they are not copied
bool aligned(const pathsig_linattn *c, const void *q, const void *k, const void *v) {
    if (copied(c) || (aligned16(q) && aligned16(k) && aligned16(v))) return true;
    set_error("q, k and v must start at multiples of 16 bytes");
    return false;
}

template <typename T>
int forward_t(const pathsig_linattn *c, const void *q, const void *k, const void *v, const float *state, void *out, float *final_state,
              char *ws, hipStream_t stream) {
    Sweep a = sweep_of(c);
    const Inputs in = inputs<T>(c, q, k, v, ws, false, stream);
    a.q = in.q;
    a.k = in.k;
    a.v = in.v;
    a.first = state;
    a.last = final_state;
    a.out = out;
    a.out_scale = c->scale;
    a.exact_state = final_state || c->learned_decay;
    float *const starts = (float *)(ws + forward_layout(c).starts);
    if (state && state == final_state && a.pieces > 1 && a.pieces <= kJoinInside) {
        const int64_t n = c->B * c->H * c->Dk * c->Dv;  // the first entry of `starts`, which only more pieces fill
        copy_state_kernel<<<(unsigned)std::min<int64_t>(ceil_div(n, 256), 4096), 256, 0, stream>>>(state, starts, n);
        a.first = starts;
    }
    fold<T>(a, starts, stream);
    chunks<T>(a, false, stream);
    return launch_status("linear attention");
}

struct BackwardLayout {
    size_t forward, ends, grad_out, wide_k, wide_v, decay, total;  // byte offsets
};

int64_t decay_partials(const pathsig_linattn *c) {
    int64_t piece;
    int pieces, run;
    cut(c, &piece, &pieces, &run);
    return pieces / run * ceil_div(c->Dk, 128) * ceil_div(c->Dv, 128) * c->B;
}

BackwardLayout backward_layout(const pathsig_linattn *c, bool want_decay) {
    BackwardLayout l = {};
    const size_t tokens = (size_t)c->B * c->L * c->H;
    l.forward = place(l.total, forward_layout(c).total);
    l.ends = place(l.total, starts_bytes(c));
    if (padded(c, c->Dv) != c->Dv) l.grad_out = place(l.total, tokens * padded(c, c->Dv) * element_of(c));
    if (c->H != c->Hkv) {
        l.wide_k = place(l.total, tokens * c->Dk * sizeof(float));
        l.wide_v = place(l.total, tokens * c->Dv * sizeof(float));
    }
    if (want_decay) l.decay = place(l.total, (size_t)decay_partials(c) * c->H * sizeof(float));
    return l;
}

// the same states with rows and columns exchanged, for the answers of a sweep alone
Sweep transposed(Sweep a) {
    std::swap(a.Dk, a.Dv);
    std::swap(a.Kp, a.Vp);
    std::swap(a.row, a.column);
    a.last = nullptr;
    a.exact_state = 0;
    return a;
}

template <typename T>
int backward_t(const pathsig_linattn *c, const void *q, const void *k, const void *v, const float *state, const char *kept,
               const void *grad_out, const float *grad_final, void *grad_q, void *grad_k, void *grad_v, float *grad_decay,
               float *grad_state, char *ws, hipStream_t stream) {
    const int64_t group = c->H / c->Hkv;
    const BackwardLayout l = backward_layout(c, grad_decay != nullptr);
    char *const from_forward = kept ? const_cast<char *>(kept) : ws + l.forward;
    const Inputs in = inputs<T>(c, q, k, v, from_forward, kept != nullptr, stream);
    const View vq = in.q, vk = in.k, vv = in.v;
    View vdo = dense(grad_out, c->L, c->H, c->Dv, 1);
    if (const int64_t V = padded(c, c->Dv); V != c->Dv) {
        const Copy one = {grad_out, ws + l.grad_out, vdo.sb, vdo.st, vdo.sh, (int)c->H, (int)c->Dv, (int)V};
        copy<T>(c, &one, 1, stream);
        vdo = dense(ws + l.grad_out, c->L, c->H, V, 1);
    }
    // the forward's states in front of the pieces
    Sweep forward = sweep_of(c);
    forward.q = vq;
    forward.k = vk;
    forward.v = vv;
    forward.first = state;
    forward.out_scale = c->scale;
    forward.exact_state = grad_decay != nullptr;
    if (kept)
        forward.starts = (float *)from_forward;
    else if (grad_q || grad_decay)
        fold<T>(forward, (float *)from_forward, stream);
    // dq: the forward with (do, v, k) and the transposed states
    if (grad_q) {
        Sweep a = transposed(forward);
        a.q = vdo;
        a.k = vv;
        a.v = vk;
        a.out = grad_q;
        chunks<T>(a, false, stream);
    }
    // dv: backwards in time with (k, q, do)
    Sweep back = sweep_of(c);
    back.q = vk;
    back.k = vq;
    back.v = vdo;
    back.first = grad_final;
    back.last = grad_state;
    back.in_scale = c->scale;
    back.reverse = 1;
    back.out_float = group > 1;
    back.out = group > 1 ? (void *)(ws + l.wide_v) : grad_v;
    back.exact_state = grad_state || grad_decay;
    if (grad_k || grad_v || grad_state || grad_decay) fold<T>(back, (float *)(ws + l.ends), stream);
    const int64_t rows = c->B * c->L;
    auto sum_heads = [&](size_t wide, void *out, int64_t D) {
        if (group == 1 || rows == 0) return;
        const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(rows * c->Hkv * D, 256), 4096);
        group_sum_kernel<T><<<blocks, 256, 0, stream>>>((const float *)(ws + wide), (T *)out, rows, (int)c->Hkv, (int)group, (int)D);
    };
    if (grad_v || grad_state) {
        back.exact_state = grad_state != nullptr;
        chunks<T>(back, false, stream);
        sum_heads(l.wide_v, grad_v, c->Dv);
    }
    // dk: backwards in time with (v, do, q), from the same states, transposed
    if (grad_k) {
        Sweep a = transposed(back);
        a.q = vv;
        a.k = vdo;
        a.v = vq;
        a.out = group > 1 ? (void *)(ws + l.wide_k) : grad_k;
        chunks<T>(a, false, stream);
        sum_heads(l.wide_k, grad_k, c->Dk);
    }
    if (grad_decay) {
        decay<T>(forward, back, vdo, (float *)(ws + l.decay), stream);
        decay_sum_kernel<<<(unsigned)c->H, 64, 0, stream>>>((const float *)(ws + l.decay), decay_partials(c), (int)c->H, grad_decay);
    }
    return launch_status("linear attention, backward");
}

template <typename T>
int step_t(const pathsig_linattn *c, const void *q, const void *k, const void *v, float *state, void *out, hipStream_t stream) {
    Sweep a = sweep_of(c);
    const int64_t group = c->H / c->Hkv;
    a.q = view(q, c->q_stride, 1);
    a.k = view(k, c->k_stride, group);
    a.v = view(v, c->v_stride, group);
    a.out = out;
    a.out_scale = c->scale;
    const dim3 grid((unsigned)c->H, (unsigned)c->B);
    const int vec = c->Dv % 4 == 0 && aligned16(state) ? 4 : 1;
    int tx_log2 = 0;
    while (tx_log2 < 6 && ((int64_t)vec << tx_log2) < c->Dv) ++tx_log2;
    if (vec == 4)
        step_kernel<T, 4><<<grid, 256, 0, stream>>>(a, state, tx_log2);
    else
        step_kernel<T, 1><<<grid, 256, 0, stream>>>(a, state, tx_log2);
    return launch_status("linear attention, step");
}

}  // namespace
}  // namespace seq
}  // namespace psig

using namespace psig;
using namespace psig::seq;

extern "C" {

size_t pathsig_linattn_forward_workspace(const pathsig_linattn *call) {
    if (check_call(call) != PATHSIG_OK) return 0;
    return forward_layout(call).total;
}

int pathsig_linattn_forward(const pathsig_linattn *call, const void *q, const void *k, const void *v, const float *state,
                            void *out, float *final_state, void *workspace, size_t workspace_bytes, void *stream) {
    if (const int rc = check_call(call)) return rc;
    if (call->B == 0) return PATHSIG_OK;
    if (call->L > 0 && (!q || !k || !v || !out)) {
        set_error("q, k, v and out must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    const size_t need = pathsig_linattn_forward_workspace(call);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        set_error("linear attention: workspace of %zu bytes needed, got %zu", need, workspace ? workspace_bytes : (size_t)0);
        return PATHSIG_ERR_WORKSPACE;
    }
    if (!aligned(call, q, k, v)) return PATHSIG_ERR_ARGUMENT;
    if (call->dtype == PATHSIG_F32) return forward_t<float>(call, q, k, v, state, out, final_state, (char *)workspace, (hipStream_t)stream);
    return forward_t<bf16>(call, q, k, v, state, out, final_state, (char *)workspace, (hipStream_t)stream);
}

size_t pathsig_linattn_backward_workspace(const pathsig_linattn *call, int want_log_decay) {
    if (check_call(call) != PATHSIG_OK) return 0;
    return backward_layout(call, want_log_decay != 0).total;
}

int pathsig_linattn_backward(const pathsig_linattn *call, const void *q, const void *k, const void *v, const float *state,
                             const void *kept, size_t kept_bytes, const void *grad_out, const float *grad_final_state, void *grad_q,
                             void *grad_k, void *grad_v, float *grad_log_decay, float *grad_state, void *workspace,
                             size_t workspace_bytes, void *stream) {
    if (const int rc = check_call(call)) return rc;
    if (call->B > 0 && call->L > 0 && (!q || !k || !v || !grad_out)) {
        set_error("q, k, v and grad_out must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (call->B > 0 && call->L > 0 && grad_state && !grad_v) {
        set_error("grad_state comes with grad_v, which must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (grad_log_decay && !call->learned_decay) {
        set_error("grad_log_decay is asked for, but learned_decay is not set");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (grad_state && (grad_state == grad_final_state || grad_state == state)) {
        set_error("grad_state must not be the buffer of grad_final_state or state, which are read after it is written");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (kept && kept_bytes != forward_layout(call).total) {
        set_error("kept: the forward's workspace has %zu bytes, got %zu", forward_layout(call).total, kept_bytes);
        return PATHSIG_ERR_ARGUMENT;
    }
    const size_t need = backward_layout(call, grad_log_decay != nullptr).total;
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        set_error("linear attention backward: workspace of %zu bytes needed, got %zu", need, workspace ? workspace_bytes : (size_t)0);
        return PATHSIG_ERR_WORKSPACE;
    }
    if (call->B == 0) {
        if (!grad_log_decay) return PATHSIG_OK;
        decay_sum_kernel<<<(unsigned)call->H, 64, 0, (hipStream_t)stream>>>(nullptr, 0, (int)call->H, grad_log_decay);
        return launch_status("linear attention, backward");
    }
    if (!aligned(call, q, k, v) || (padded(call, call->Dv) == call->Dv && !aligned16(grad_out))) {
        set_error("q, k, v and grad_out must start at multiples of 16 bytes");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (call->dtype == PATHSIG_F32)
        return backward_t<float>(call, q, k, v, state, (const char *)kept, grad_out, grad_final_state, grad_q, grad_k, grad_v,
                                 grad_log_decay, grad_state, (char *)workspace, (hipStream_t)stream);
    return backward_t<bf16>(call, q, k, v, state, (const char *)kept, grad_out, grad_final_state, grad_q, grad_k, grad_v,
                            grad_log_decay, grad_state, (char *)workspace, (hipStream_t)stream);
}

int pathsig_linattn_step(const pathsig_linattn *call, const void *q, const void *k, const void *v, float *state, void *out,
                         void *stream) {
    if (const int rc = check_call(call)) return rc;
    if (call->L != 1 || call->lengths) {
        set_error("a step has one token of every sequence: L must be 1 and lengths NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (call->B == 0) return PATHSIG_OK;
    if (!q || !k || !v || !state || !out) {
        set_error("q, k, v, state and out must not be NULL");
        return PATHSIG_ERR_ARGUMENT;
    }
    if (call->dtype == PATHSIG_F32) return step_t<float>(call, q, k, v, state, out, (hipStream_t)stream);
    return step_t<bf16>(call, q, k, v, state, out, (hipStream_t)stream);
}

}  // extern "C"
