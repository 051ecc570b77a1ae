// Sweeps of linear attention over whole sequences: what the entry points (seq_attention.hip) and the kernels of the chunked form
// (seq_chunks.hip, compiled once for each width of the keys) share.
#pragma once

#include "seq_common.hpp"

namespace psig {
namespace seq {

// A [B, L, heads, D] tensor; heads[h / group] is read for head h.  Rows start at multiples of 16 bytes and hold whole units of 16
// bytes: tensors that do not lie so are copied first, with zeros behind the last channel.
struct View {
    const void *p;
    int64_t sb, st, sh;
    int group;
};

constexpr float kLog2e = 1.44269504088896340736f;

// One pass of the recurrence over all tokens, S <- decay S + in_scale k v^T, out = out_scale S^T q, or backwards in time, where
// the decay comes after the token: S <- S + in_scale k v^T, out = out_scale S^T q, S <- decay S.  Dk and Dv are the rows and
// columns of this pass' state, whichever tensors are in the places of k and v.
struct Sweep {
    View q, k, v;
    // [B, H, Dk * Dv], each may be NULL: the state in front of the first token, whose element (a, c) lies at a * row + c * column
    // of a head's (as in `starts`), and the one behind the last, row by row
    const float *first;
    float *last;
    int64_t row, column;
    void *out;             // [B, L, H, Dv] dense
    int out_float;         // float32 instead of the type of q
    const float *log_decay;
    const int32_t *lengths;
    int64_t B, L;
    int H, Dk, Dv, Kp, Vp;  // Kp, Vp: channels of a row of q and k, and of v, in whole units
    float in_scale, out_scale;
    int reverse;
    int exact_state;       // the state is wanted in 32 bits, not only the answers
    // the sequence in pieces of `piece` tokens: starts [pieces][B][H][Dk * Dv], whose s-th entry is the state in front of piece s
    // or, with few pieces (kJoinInside), what piece s - 1 adds to a state of zero.  A block of the sweep takes `run` of them, one
    // after the other.
    int64_t piece;
    int pieces, run;
    float *starts;
};

// Up to so many pieces, every block adds up the pieces before its own by itself: at most 1.5 states read for each block instead of
// a launch that reads all of them and writes them back (measured with two pieces of 256 heads, 128 x 128: 25 us).
constexpr int kJoinInside = 4;

__device__ __forceinline__ int64_t length_of(const int32_t *lengths, int64_t b, int64_t L) {
    if (!lengths) return L;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > L ? L : n;
}

__device__ __forceinline__ float decay_of(const float *log_decay, int h) {
    // (minus infinity forgets everything at once; a finite stand-in keeps 0 * g at 0.  NaN stays)
    const float g = log_decay[h];
    return g < -1e30f ? -1e30f : g;
}

// Tokens [begin, end) of `count` pieces from the s-th on, in the order of the sweep.  Pieces are cut at the same tokens in both
// directions of time: the s-th of a sweep backwards in time is the one s from the last, and empty where the sequence ends
// before it.
struct Range {
    int64_t begin, end;
};
__device__ __forceinline__ Range range_of(const Sweep &a, int64_t n, int s, int count = 1) {
    const int64_t p = a.reverse ? a.pieces - s - count : s;
    const int64_t t0 = min(p * a.piece, n), t1 = min((p + count) * a.piece, n);
    return a.reverse ? Range{n - t1, n - t0} : Range{t0, t1};
}

// seq_chunks.hip, for keys of up to 32 DKT channels.  fold: only the states that the pieces add, from zero, into starts[s + 1].
template <typename T, int DKT>
void launch_chunks(const Sweep &a, bool fold, hipStream_t stream);

// The gradient of the decays: partial sums [runs][slices][B][H], slices = decay_slices().  a: the sweep forwards in time; back: the
// one backwards in time with the same rows and columns, whose states are the gradients of a's.
inline int decay_slices(const Sweep &a) { return (int)(ceil_div(a.Dk, 128) * ceil_div(a.Dv, 128)); }
template <typename T, int DKT>
void launch_decay(const Sweep &a, const Sweep &back, const View &grad_out, float *partial, hipStream_t stream);

}  // namespace seq
}  // namespace psig
