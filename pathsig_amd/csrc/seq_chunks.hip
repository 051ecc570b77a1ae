// Linear attention over whole sequences in chunks, on matrix instructions.
//
// In a chunk of C tokens that starts from the state S, with l = e^g and token i of the chunk counted from 0:
//     o_i = l^(i+1) S^T q_i + sum over j <= i of l^(i-j) (q_i . k_j) v_j,
//     S' = l^C S + sum over j of l^(C-1-j) k_j v_j^T.
// Backwards in time the decay comes after the token: exponents i and C - j in place of i + 1 and C - 1 - j.
//
// A block has a head of a sequence (or of a piece of it) and up to 128 columns of its state; wave w has the 32 columns from
// 32 w on, its part of the state in accumulator registers from the first chunk to the last.  All products are 32 x 32 tiles
// laid out so that little crosses lanes:
//   * scores transposed, K Q^T: a lane has one token i and sixteen j.  Decays and the causal mask are then factors of a lane's
//     registers, and the rounded scores are, as they stand, the right operand of V^T P.  The tiles are dealt to the waves (a single
//     tile: its channels) and exchanged through LDS; computed by every wave they took a quarter of the matrix instructions;
//   * answers transposed, S^T Q^T + V^T P: the state's accumulators, rounded, are, as they stand, the left operand;
//   * an accumulator holds rows 8 (r / 4) + 4 (lane / 32) + r % 4.  Operands are read in that order of the contracted index
//     ("accumulator order"): Q and K rows from LDS, where the channels of 16 are stored so that a lane's eight lie side by side,
//     V^T and K^T with transposing reads of four rows each.
// A chunk takes two barriers: before the first its tiles are stored, from registers that were loaded while the chunk before was
// worked on; between the two everything that reads tiles happens; after the second the next chunk's tiles are stored while the
// answers are finished from registers and scores.
//
// Rounding in bf16: scores and the state's copy for the products with V and Q are split into two terms of bf16 each, which are off by
// 2^-16 of them: an answer is rounded once, at its end.  (With one term they are off by as much as that rounding: root mean square
// of the error 2.35e-3 of the answers against 1.66e-3; a sweep of 16 x 4096 tokens of 16 heads of 128 took 270 us with one and
// takes 310 with two.)  The state itself stays in 32 bits, and so does what is added to it: l^(C-1-j) v_j is split too, three terms hold all
// 24 bits (launch_terms).
//
// A first chunk that is not full is filled from the front with tokens of zeros, so that the factors l^(C-1-j) hold for every
// chunk and none of them is a quotient.
//
// Bound by memory first: 16 x 4096 tokens of 16 heads of 128 in bf16 are 1.07 GB to read and write, 210 us at the rate of a large
// copy (5.1 TB/s); the sweep takes 310 in two pieces, two blocks to a compute unit with 48 KB each on their way.  What two waves to a
// SIMD do not hide: 76 to 84 matrix instructions and about 790 vector ones a chunk and wave (a quarter of the time each), one after
// the other between two barriers, and 24 of 256 registers that are spilled.  In one piece, one block to a unit, it took 356 where two
// took 290.
#include <algorithm>

#include "seq_attention.hpp"

namespace psig {
namespace seq {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// eight elements of an operand, a lane's share of sixteen steps of the contracted index
template <typename T>
struct FragOf;
template <>
struct FragOf<bf16> {
    using type = bf16x8;
};
template <>
struct FragOf<float> {
    using type = f32x8;
};
template <typename T>
using Frag = typename FragOf<T>::type;

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

template <typename T>
__device__ __forceinline__ Frag<T> rounded(f32x8 x) {
    return __builtin_convertvector(x, Frag<T>);
}
__device__ __forceinline__ f32x8 widened(bf16x8 x) { return __builtin_convertvector(x, f32x8); }
__device__ __forceinline__ f32x8 widened(f32x8 x) { return x; }

template <int Half>
__device__ __forceinline__ f32x8 half_of(f32x16 x) {
    if constexpr (Half == 0)
        return __builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, 6, 7);
    else
        return __builtin_shufflevector(x, x, 8, 9, 10, 11, 12, 13, 14, 15);
}

// the same in all lanes, in a scalar register
__device__ __forceinline__ float uniform(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// row of accumulator register r
__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

// A tile of rows of D channels in LDS, in units of 16 bytes.  Units of a row are exchanged by a pattern of the row number: rows
// read at one unit by 16 lanes, and four neighbouring rows read at 64 neighbouring bytes (the transposing reads), each fall
// into different banks.  The pattern repeats after 16 rows, so every address is a lane's base, exclusive-or a constant, plus a
// constant.
template <typename T, int D>
struct Tile;

template <int D>
struct Tile<bf16, D> {
    static constexpr int kUnits = D / 8, kPerUnit = 8, kRow = D * 2, kColumnBases = 2;
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (kUnits >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        if constexpr (kUnits == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        return (row >> 2) & 3;
    }
    // Channels of a group of sixteen are stored in fours as 0, 2 | 1, 3: a unit is what one half of the lanes contracts
    static __device__ __forceinline__ void store(char *lds, int row, int unit, u32x4 x) {
        const int at = row * kRow + (((unit & ~1) ^ swizzle(row)) * 16) + (unit & 1) * 8;
        *(u32x2 *)(lds + at) = u32x2{x[0], x[1]};
        *(u32x2 *)(lds + (at ^ 16)) = u32x2{x[2], x[3]};
    }
    static __device__ __forceinline__ int row_base(int ln, int half) { return ln * kRow + ((half ^ swizzle(ln)) * 16); }
    // channels 16 kk .. 16 kk + 15 of row 32 tile + lane % 32, in accumulator order
    static __device__ __forceinline__ bf16x8 row(const char *lds, int base, int tile, int kk) {
        return *(const bf16x8 *)(lds + (base ^ (kk * 32)) + tile * 32 * kRow);
    }
    // (a group of sixteen lanes reads four rows of sixteen channels, each lane four channels of one row, and gets four rows of one
    // channel)
    static __device__ __forceinline__ void column_bases(int (&base)[kColumnBases], int lane) {
        const int half = lane >> 5, part = (lane >> 4) & 1, r = (lane & 15) >> 2, four = lane & 3;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int j = 8 * g + 4 * half + r;
            base[g] = j * kRow + (((2 * part + (four & 1)) ^ swizzle(j)) * 16) + (four >> 1) * 8;
        }
    }
    // channel 32 m + lane % 32 of rows 16 kk .. 16 kk + 15, in accumulator order
    static __device__ __forceinline__ bf16x8 column(const char *lds, const int (&base)[kColumnBases], int m, int kk) {
        s16x4 got[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char *const p = lds + (base[g] ^ (m * 64)) + kk * 16 * kRow;
            got[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
        }
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(got[0], got[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

template <int D>
struct Tile<float, D> {
    static constexpr int kUnits = D / 4, kPerUnit = 4, kRow = D * 4, kColumnBases = 1;
    static __device__ __forceinline__ constexpr int swizzle(int row) {
        return (((row & 4) << 1) | ((row & 8) >> 1) | (row & 3)) & (kUnits - 1);
    }
    static __device__ __forceinline__ void store(char *lds, int row, int unit, u32x4 x) {
        *(u32x4 *)(lds + row * kRow + ((unit ^ swizzle(row)) * 16)) = x;
    }
    static __device__ __forceinline__ int row_base(int ln, int half) { return ln * kRow + ((half ^ swizzle(ln)) * 16); }
    static __device__ __forceinline__ f32x8 row(const char *lds, int base, int tile, int kk) {
        const f32x4 a = *(const f32x4 *)(lds + (base ^ (kk * 64)) + tile * 32 * kRow);
        const f32x4 b = *(const f32x4 *)(lds + (base ^ (kk * 64 + 32)) + tile * 32 * kRow);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ void column_bases(int (&base)[kColumnBases], int lane) {
        const int ln = lane & 31, half = lane >> 5;
        base[0] = 4 * half * kRow + (((ln >> 2) ^ swizzle(4 * half)) * 16) + (ln & 3) * 4;
    }
    static __device__ __forceinline__ f32x8 column(const char *lds, const int (&base)[kColumnBases], int m, int kk) {
        f32x8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int j = acc_row(e, 0);
            x[e] = *(const float *)(lds + (base[0] ^ (m * 128) ^ (swizzle(j) * 16)) + (16 * kk + j) * kRow);
        }
        return x;
    }
};

// The units of a tile of ROWS rows that one of THREADS threads fetches: registers between the load from memory and the store to
// LDS.
template <typename T, int D, int ROWS, int THREADS>
struct Fetch {
    using L = Tile<T, D>;
    static constexpr int kTotal = ROWS * L::kUnits, kEach = (kTotal + THREADS - 1) / THREADS;
    static constexpr int kRowsApart = THREADS / L::kUnits;  // rows between a thread's units
    static_assert(THREADS % L::kUnits == 0, "a thread's units lie in one column");
    u32x4 x[kEach];

    // p: the tile's first row and channel.  The rows before `pad` are zeros and not read, as are channels from `channels` on, a
    // multiple of a unit.  st: from row to row, backwards in time negative.
    __device__ __forceinline__ void load(const T *p, int st, int channels, int pad) {
        const int row0 = threadIdx.x / L::kUnits, c = threadIdx.x % L::kUnits * L::kPerUnit;
        const int offset = row0 * st + c;
        if (kTotal % THREADS == 0 && pad <= 0 && channels >= D) {
#pragma unroll
            for (int u = 0; u < kEach; ++u) x[u] = *(const u32x4 *)(p + (int64_t)u * kRowsApart * st + offset);
            return;
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int row = row0 + u * kRowsApart;
            x[u] = u32x4{0, 0, 0, 0};
            if ((kTotal % THREADS && row >= ROWS) || row < pad || c >= channels) continue;
            x[u] = *(const u32x4 *)(p + (int64_t)u * kRowsApart * st + offset);
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
        const int row0 = threadIdx.x / L::kUnits, unit = threadIdx.x % L::kUnits;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int row = row0 + u * kRowsApart;
            if (kTotal % THREADS && row >= ROWS) continue;
            L::store(lds, row, unit, x[u]);
        }
    }
};

// x - hi of eight elements, hi being x rounded: exact, a product with minus one added in 32 bits.  Where hi is infinite or no number
// the remainder, and that of the element beside it, is zero (the median of NaN, zero and NaN), so that an infinity is not taken
// from itself.
__device__ __forceinline__ f32x8 remainder(f32x8 x, bf16x8 hi) {
    uint32_t low = 0xbf80u, high = 0xbf800000u;  // minus one beside zero
    asm("" : "+s"(low), "+s"(high));             // (in registers: as an inline constant the compiler puts it into both halves)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const bf16x2 pair = {hi[e], hi[e + 1]};
        x[e] = __builtin_amdgcn_fdot2_f32_bf16(pair, __builtin_bit_cast(bf16x2, low), x[e], false);
        x[e + 1] = __builtin_amdgcn_fdot2_f32_bf16(pair, __builtin_bit_cast(bf16x2, high), x[e + 1], false);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_fmed3f(x[e], 0.f, x[e]);
    return x;
}

// x in COUNT terms of the type of the products; three of bf16 hold all 24 bits
template <typename T, int COUNT>
__device__ __forceinline__ void split(f32x8 x, Frag<T> (&out)[COUNT]) {
    out[0] = rounded<T>(x);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 1; i < COUNT; ++i) {
            x = remainder(x, out[i - 1]);
            out[i] = rounded<T>(x);
        }
    }
}

// f x in terms
template <typename T, int COUNT>
__device__ __forceinline__ void split_scaled(f32x8 x, const f32x8 &f, Frag<T> (&out)[COUNT]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f[e];
    split<T>(x, out);
}

// Bytes that a thread fetches of a chunk of 32 tiles tokens.
constexpr int fetched(int element, int tiles, int DKT, int NW) { return 32 * tiles * (2 * 32 * DKT + 32 * NW) * element / (64 * NW); }

// 64 tokens in bf16, half as many where a thread would fetch more than 320 bytes of a chunk, and in fp32, where it is twice as
// many bytes
template <typename T>
constexpr int chunk_tiles(int DKT, int NW) {
    return sizeof(T) == 2 && fetched(2, 2, DKT, NW) <= 320 ? 2 : 1;
}

// The state in front of a piece (FOLD: zero): this lane's column dv, rows in accumulator order.
template <int DKT, int NW, bool FOLD>
__device__ __forceinline__ void load_state(f32x16 (&S)[DKT], const Sweep &a, int64_t b, int h, int64_t n, int piece, float g2, int dk0,
                                           int dv0, int dv, int half) {
    const int64_t plane = (int64_t)a.Dk * a.Dv, head = (b * a.H + h) * plane, between = a.B * a.H * plane;
#pragma unroll
    for (int t = 0; t < DKT; ++t) S[t] = f32x16{};
    if (FOLD) return;
    const bool joined = a.pieces > kJoinInside, whole = dk0 + 32 * DKT <= a.Dk && dv0 + 32 * NW <= a.Dv;
    const int row = (int)a.row, column = (int)a.column;
    // one base for all lanes and 32-bit offsets; rows and columns behind the last are zeros, their addresses are kept inside
    const uint32_t offset = whole ? dv * column + (dk0 + 4 * half) * row : min(dv, a.Dv - 1) * column;
    // the state in front of the first token (s = -1) and what the pieces up to this one add, or all of that at once
    const int s0 = joined ? piece - 1 : a.first ? -1 : 0;
    for (int s = s0; s < piece; ++s) {
        const float *const p = (s < 0 && !joined ? a.first : a.starts + (s + 1) * between) + head;
        float f = 0.f;  // (of the zeros in front of the first, whatever the decay)
        if (s > s0) {
            const Range r = range_of(a, n, s);
            f = exp2f(g2 * (float)(r.end - r.begin));
        }
        f32x16 x[DKT];  // (all loads are on their way before the first is waited for)
        if (whole && row == 1) {
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    float four[4];
                    __builtin_memcpy(four, p + 32 * t + 8 * r4 + offset, 16);  // (a state may start at any float)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[t][4 * r4 + e] = four[e];
                }
        } else if (whole) {
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[t][r] = (p + (32 * t + acc_row(r, 0)) * row)[offset];
        } else {
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int dk = dk0 + 32 * t + acc_row(r, half);
                    const float y = p[offset + (uint32_t)(min(dk, a.Dk - 1) * row)];
                    x[t][r] = dk < a.Dk && dv < a.Dv ? y : 0.f;
                }
        }
#pragma unroll
        for (int t = 0; t < DKT; ++t) S[t] = S[t] * f + x[t];
    }
}

// CT: tiles of 32 tokens to a chunk.  TERMS: of l^(C-1-j) v_j in the state's update.
template <typename T, typename O, int DKT, int NW, int CT, int TERMS, bool FOLD>
__global__ __launch_bounds__(64 * NW, DKT <= 4 && NW >= DKT ? 2 : 1) void chunk_kernel(const Sweep a, int slices) {
    constexpr int DK = 32 * DKT, DV = 32 * NW, C = 32 * CT, THREADS = 64 * NW;
    // fetched a chunk ahead, where registers allow it
    constexpr bool kAhead = fetched(sizeof(T), CT, DKT, NW) <= 320;
    // Scores: tiles (j, i) = (0, 0), (0, 1), (1, 1) are dealt to the waves; a single tile is split along the channels instead
    constexpr int kTiles = CT * (CT + 1) / 2, kParts = CT == 1 ? (NW < 2 * DKT ? NW : 2 * DKT) : 1, kSteps = DK / 16 / kParts;
    using KTile = Tile<T, DK>;
    using VTile = Tile<T, DV>;
    constexpr int kKBytes = C * KTile::kRow, kVBytes = C * VTile::kRow;
    __shared__ __align__(16) char lds[kKBytes * (FOLD ? 1 : 2) + kVBytes];
    // Tables of factors.  The small ones lie where that of the diagonal tiles has the last four j of too small an i, which nothing reads:
    // with them beside it a block of 64 x 64 would have 384 bytes too many for four blocks to a compute unit.
    __shared__ __align__(16) f32x4 table_diagonal[FOLD ? 1 : 4][64];
    f32x4 (&table_left)[CT][4][2] = *(f32x4 (*)[CT][4][2])&table_diagonal[FOLD ? 0 : 3][32];
    f32x4 (&table_later)[4][2] = *(f32x4 (*)[4][2])&table_diagonal[FOLD ? 0 : 3][32 + 8 * CT];
    constexpr int kSmall = 8 * CT + 8;
    static_assert(kSmall <= 28, "the unit of (r / 4, lane) = (3, 32 + i) has j = 28 .. 31 of token i");
    // scores as operands, in terms (a wave alone keeps them), or the parts of a tile's sums
    constexpr int kTerms = sizeof(T) == 2 ? 2 : 1;
    __shared__ __align__(16) Frag<T> scores[FOLD || kParts > 1 || NW == 1 ? 1 : kTiles][2][kTerms][64];
    __shared__ __align__(16) f32x4 sums[!FOLD && kParts > 1 ? kParts : 1][4][64];
    char *const lds_k = lds, *const lds_v = lds + kKBytes, *const lds_q = lds_v + kVBytes;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, ln = lane & 31;
    const int slice = blockIdx.x % slices, h = blockIdx.x / slices, run = FOLD ? 1 : a.run, piece = blockIdx.y * run;
    const int64_t b = blockIdx.z;
    const int dv0 = slice * DV, dv = dv0 + 32 * wave + ln;  // this lane's column of the state
    const int64_t n = length_of(a.lengths, b, a.L);
    const auto [begin, end] = range_of(a, n, piece, run);
    const float g2 = decay_of(a.log_decay, h) * kLog2e;
    const int64_t plane = (int64_t)a.Dk * a.Dv, head = (b * a.H + h) * plane;

    if (!FOLD) {
        // tokens behind the end of the sequence
        const int64_t p = a.reverse ? a.pieces - piece - run : piece;
        const int64_t z0 = max(n, p * a.piece), z1 = min((p + run) * a.piece, a.L);
        const int width = min(DV, a.Dv - dv0);
        for (int64_t t = z0 + wave; t < z1; t += NW)
            for (int c = lane; c < width; c += 64) ((O *)a.out)[((b * a.L + t) * a.H + h) * a.Dv + dv0 + c] = from_float<O>(0.f);
    }
    const bool owns_end = !FOLD && a.last && end == n && (begin < n || (n == 0 && piece == 0));
    if (begin >= end && !owns_end && !FOLD) return;

    f32x16 S[DKT];
    load_state<DKT, NW, FOLD>(S, a, b, h, n, piece, g2, 0, dv0, dv, half);

    const int chunks = (int)((max(end - begin, (int64_t)0) + C - 1) / C);
    int64_t r0 = end - (int64_t)chunks * C;  // of the chunk being worked on; before `begin` where the first is not full
    // A decay above 1 may have powers that overflow where a chunk is full, and would make NaN of the zeros of padding.  A single chunk
    // has no factors for tokens of padding and for gaps that no two of its tokens have, and a state of zeros in front of it stays one.
    // (Behind a padded chunk, a full one has those gaps.)
    const bool grows = g2 > 0.f && chunks == 1;
    const int padded = grows ? (int)(begin - r0) : 0, most = C - padded;
    const float g_state = uniform(grows && (FOLD || (piece == 0 && !a.first)) ? 0.f : g2);

    // Factors of a lane's registers, in LDS (they would fill the registers, and are read once a chunk): l^(C - 1 - j) for the state's
    // update; for scores l^(31 - j), which l^(i + 1) completes in the tile off the diagonal, and l^(i - j) in those on it (j after i
    // is masked where it is used)
    const float both = a.in_scale * a.out_scale;
    if (threadIdx.x < 64) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = acc_row(r, half);
            if (ln == 0) {
                table_later[r / 4][half][r % 4] = j < padded ? 0.f : exp2f(g2 * (float)(31 - j));
#pragma unroll
                for (int t = 0; t < CT; ++t)
                    table_left[t][r / 4][half][r % 4] =
                        32 * t + j < padded ? 0.f : a.in_scale * exp2f(g2 * (float)(C - 1 - 32 * t - j + a.reverse));
            }
            if constexpr (!FOLD) {
                if (r < 12 || lane < 32 || ln >= kSmall)
                    table_diagonal[r / 4][lane][r % 4] = ln - j < most ? both * exp2f(g2 * (float)max(ln - j, 0)) : 0.f;
            }
        }
    }
    const float since = ln + 1 < most ? both * exp2f(g2 * (float)(ln + 1)) : 0.f;

    const T *const kp = (const T *)a.k.p + b * a.k.sb + (h / a.k.group) * a.k.sh;
    const T *const vp = (const T *)a.v.p + b * a.v.sb + (h / a.v.group) * a.v.sh + dv0;
    const T *const qp = FOLD ? nullptr : (const T *)a.q.p + b * a.q.sb + (h / a.q.group) * a.q.sh;
    const int sign = a.reverse ? -1 : 1;
    Fetch<T, DK, C, THREADS> fk, fq;
    Fetch<T, DV, C, THREADS> fv;
    // (where registers do not hold a whole chunk, the tensors pass through them one after the other)
    auto fetch = [&](int64_t at, int pad) {
        const int64_t t = a.reverse ? n - 1 - at : at;
        fk.load(kp + t * a.k.st, sign * (int)a.k.st, a.Kp, pad);
        if (!kAhead) fk.store(lds_k);
        fv.load(vp + t * a.v.st, sign * (int)a.v.st, a.Vp - dv0, pad);
        if (!kAhead) fv.store(lds_v);
        if (!FOLD) fq.load(qp + t * a.q.st, sign * (int)a.q.st, a.Kp, pad);
        if (!kAhead && !FOLD) fq.store(lds_q);
    };
    auto store = [&]() {
        fk.store(lds_k);
        fv.store(lds_v);
        if (!FOLD) fq.store(lds_q);
    };
    if (chunks > 0) {
        fetch(r0, (int)(begin - r0));
        if (kAhead) {
            store();
            if (chunks > 1) fetch(r0 + C, 0);
        }
    }
    const int row_base_of_lane = KTile::row_base(ln, half);
    int k_bases_of_lane[KTile::kColumnBases], v_bases_of_lane[VTile::kColumnBases];
    KTile::column_bases(k_bases_of_lane, lane);
    VTile::column_bases(v_bases_of_lane, lane);
    for (int c = 0; c < chunks; ++c, r0 += C) {
        const int pad = (int)max(begin - r0, (int64_t)0);
        __syncthreads();  // this chunk's tiles are in LDS, the scores of the chunk before are read

        // (addresses are worked out from these in every chunk: held for all reads, they would fill the registers)
        int row_base = row_base_of_lane, k_bases[KTile::kColumnBases], v_bases[VTile::kColumnBases];
        asm volatile("" : "+v"(row_base));
#pragma unroll
        for (int g = 0; g < KTile::kColumnBases; ++g) {
            k_bases[g] = k_bases_of_lane[g];
            v_bases[g] = v_bases_of_lane[g] ^ (wave * 32 * (int)sizeof(T));
            asm volatile("" : "+v"(k_bases[g]), "+v"(v_bases[g]));
        }

        // scores
        f32x16 out[FOLD ? 1 : CT];
        Frag<T> own[NW == 1 && !FOLD ? kTiles : 1][2][kTerms];
        if constexpr (!FOLD) {
            if constexpr (kParts > 1) {
                if (wave < kParts) {
                    f32x16 P = {};
                    const int base = row_base ^ (wave * kSteps * 16 * (int)sizeof(T));
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) P = mma(KTile::row(lds_k, base, 0, kk), KTile::row(lds_q, base, 0, kk), P);
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) sums[wave][r4][lane] = f32x4{P[4 * r4], P[4 * r4 + 1], P[4 * r4 + 2], P[4 * r4 + 3]};
                }
            } else {
                auto score = [&](int tile, auto keep) {
                    const int i = tile > 0, j = tile > 1;
                    f32x16 P = {};
                    const char *const kt = lds_k + j * 32 * KTile::kRow, *const qt = lds_q + i * 32 * KTile::kRow;
#pragma unroll
                    for (int kk = 0; kk < DK / 16; ++kk) P = mma(KTile::row(kt, row_base, 0, kk), KTile::row(qt, row_base, 0, kk), P);
                    if (i == j) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            // (selected, not multiplied by zero: a score of a later token may be infinite)
                            P[r] = acc_row(r, half) <= ln ? P[r] * table_diagonal[r / 4][lane][r % 4] : 0.f;
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) P[r] *= table_later[r / 4][half][r % 4] * since;
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        Frag<T> terms[kTerms];
                        split<T>(s ? half_of<1>(P) : half_of<0>(P), terms);
#pragma unroll
                        for (int e = 0; e < kTerms; ++e) keep(s, e, terms[e]);
                    }
                };
                if constexpr (NW == 1) {
#pragma unroll
                    for (int tile = 0; tile < kTiles; ++tile) score(tile, [&](int s, int e, Frag<T> x) { own[tile][s][e] = x; });
                } else {
                    for (int tile = wave; tile < kTiles; tile += NW)
                        score(tile, [&](int s, int e, Frag<T> x) { scores[tile][s][e][lane] = x; });
                }
            }
            // answers from the state
#pragma unroll
            for (int i = 0; i < CT; ++i) out[i] = f32x16{};
#pragma unroll
            for (int kk = 0; kk < DK / 16; ++kk) {
                Frag<T> st[kTerms], q[CT];
                split<T>(kk % 2 ? half_of<1>(S[kk / 2]) : half_of<0>(S[kk / 2]), st);
#pragma unroll
                for (int i = 0; i < CT; ++i) q[i] = KTile::row(lds_q, row_base, i, kk);
#pragma unroll
                for (int e = 0; e < kTerms; ++e)
#pragma unroll
                    for (int i = 0; i < CT; ++i) out[i] = mma(st[e], q[i], out[i]);
            }
        }

        // the state after the chunk
        Frag<T> vt[CT][2];
        const float whole = exp2f(g_state * (float)(C - pad));
#pragma unroll
        for (int t = 0; t < DKT; ++t) S[t] *= whole;
#pragma unroll
        for (int j = 0; j < CT; ++j) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                vt[j][s] = VTile::column(lds_v, v_bases, 0, 2 * j + s);
                f32x8 f;
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = table_left[j][2 * s + e / 4][half][e % 4];
                Frag<T> terms[TERMS];
                split_scaled<T>(widened(vt[j][s]), f, terms);
#pragma unroll
                for (int t = 0; t < DKT; ++t) {
                    const Frag<T> kt = KTile::column(lds_k, k_bases, t, 2 * j + s);
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) S[t] = mma(kt, terms[i], S[t]);
                }
            }
        }

        __syncthreads();  // the tiles are read, the scores are in LDS
        if (c + 1 < chunks) {
            if (kAhead) {
                store();
                if (c + 2 < chunks) fetch(r0 + 2 * C, 0);
            } else {
                fetch(r0 + C, 0);
            }
        }
        if constexpr (!FOLD) {
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                // (rows of padding have answers that no one reads; their exponent is kept from turning around)
                out[i] *= a.out_scale * exp2f(g_state * (float)max(32 * i + ln + 1 - a.reverse - pad, 0));
                if constexpr (kParts > 1) {
                    f32x8 P[2];
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        f32x4 x = sums[0][r4][lane];
#pragma unroll
                        for (int w = 1; w < kParts; ++w) x += sums[w][r4][lane];
                        x *= table_diagonal[r4][lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) P[r4 / 2][r4 % 2 * 4 + e] = acc_row(4 * r4 + e, half) <= ln ? x[e] : 0.f;
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        Frag<T> terms[kTerms];
                        split<T>(P[s], terms);
#pragma unroll
                        for (int e = 0; e < kTerms; ++e) out[i] = mma(vt[0][s], terms[e], out[i]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j <= i; ++j)
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int e = 0; e < kTerms; ++e)
                                out[i] = mma(vt[j][s], NW == 1 ? own[NW == 1 ? i + j : 0][s][e] : scores[NW == 1 ? 0 : i + j][s][e][lane], out[i]);
                }
                const int row = 32 * i + ln;
                if (row >= pad) {
                    const int64_t t = a.reverse ? n - 1 - (r0 + row) : r0 + row;
                    O *const to = (O *)a.out + ((b * a.L + t) * a.H + h) * a.Dv;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int d = dv0 + 32 * wave + 8 * g + 4 * half;
                        if (a.Dv % 4 == 0) {  // (rows of whole fours start at multiples of four)
                            if (d < a.Dv) {
                                Pack<O, 4> four;
#pragma unroll
                                for (int e = 0; e < 4; ++e) four.v[e] = from_float<O>(out[i][4 * g + e]);
                                *(Pack<O, 4> *)(to + d) = four;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (d + e < a.Dv) to[d + e] = from_float<O>(out[i][4 * g + e]);
                        }
                    }
                }
            }
        }
    }

    float *to = FOLD ? a.starts + (int64_t)(piece + 1) * a.B * a.H * plane : owns_end ? a.last : nullptr;
    if (!to) return;
    to += head;
    const uint32_t offset = dv + 4 * half * a.Dv;
#pragma unroll
    for (int t = 0; t < DKT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (32 * t + acc_row(r, half) < a.Dk && dv < a.Dv) (to + (32 * t + acc_row(r, 0)) * a.Dv)[offset] = S[t][r];
}

// dL/dg of a piece.  With S the state of a head and D = dS/dg (zero in front of the piece, whose own S is given):
//     dL/dg = sum over chunks of  sum over j <= i of (i - j) l^(i-j) (do_i . v_j) (q_i . k_j)
//                                 + <D, G> + <S, G'>,   G = sum of l^(i+1) q_i do_i^T,  G' = sum of (i + 1) l^(i+1) q_i do_i^T,
//             + <D behind the piece, dL/dS behind the piece>,
//     D' = l^C (D + C S) + sum of (C - 1 - j) l^(C-1-j) k_j v_j^T.
// Every term is a sum of like signs or of independent ones; sum over t of t (q_t . dq_t - k_t . dk_t), which needs no states,
// cancels by the length of the sequence over the memory of the head.  Products of states stay in 32 bits (element by element on
// accumulators); what enters them is split into three bf16 terms.
__device__ __forceinline__ float sum16(f32x16 x) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += x[r];
    return s;
}

template <typename T, int DKT, int NW>
__global__ __launch_bounds__(64 * NW, DKT == 1 || (DKT == 2 && sizeof(T) == 4) ? 2 : 1) void decay_kernel(const Sweep a, const Sweep back, const View grad, float *partial,
                                                         int slices) {
    constexpr int DK = 32 * DKT, DV = 32 * NW, THREADS = 64 * NW, TERMS = sizeof(T) == 2 ? 3 : 1;
    constexpr int CT = chunk_tiles<T>(DKT, NW), C = 32 * CT;
    // fetched a chunk ahead in bf16 (4 x 8192 tokens, 8 heads of 64 x 128: 153 -> 141 us); in fp32, whose chunks are half as long, the
    // registers it takes cost the second block on a compute unit (50 x 333, 6 heads of 40 x 56: 88 -> 115)
    constexpr bool kAhead = sizeof(T) == 2 && fetched(2, CT, DKT, NW) + C * DV * 2 / THREADS <= 256;
    using KTile = Tile<T, DK>;
    using VTile = Tile<T, DV>;
    constexpr int kKBytes = C * KTile::kRow, kVBytes = C * VTile::kRow;
    __shared__ __align__(16) char lds[2 * kKBytes + 2 * kVBytes];
    __shared__ double meet[NW];
    // Factors by token of a chunk: l^(i+1) and l^(C-1-j), and by lane and register gap l^gap / kGap in tiles on the diagonal and off it
    // (accumulator order, zero where j is not before i; kGap is above all gaps, so that no factor overflows where the power does not)
    constexpr float kGap = 64.f;
    __shared__ __align__(16) f32x4 table_since[C / 4], table_left[C / 4], table_gap[CT][4][64];
    char *const lds_k = lds, *const lds_q = lds + kKBytes, *const lds_v = lds_q + kKBytes, *const lds_o = lds_v + kVBytes;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, ln = lane & 31;
    // Rows of the state are dealt to blocks like its columns: every term is a sum over both (inside a chunk, of products of a sum over
    // rows with one over columns)
    const int slice = blockIdx.x % slices, h = blockIdx.x / slices, piece = blockIdx.y * a.run;
    const int64_t b = blockIdx.z;
    const int across = (a.Dv + DV - 1) / DV, dk0 = slice / across * DK, dv0 = slice % across * DV, dv = dv0 + 32 * wave + ln;
    const int64_t n = length_of(a.lengths, b, a.L);
    const auto [begin, end] = range_of(a, n, piece, a.run);
    const float g2 = decay_of(a.log_decay, h) * kLog2e;

    f32x16 S[DKT], D[DKT];
    load_state<DKT, NW, false>(S, a, b, h, n, piece, g2, dk0, dv0, dv, half);
#pragma unroll
    for (int t = 0; t < DKT; ++t) D[t] = f32x16{};
    const T *const kp = (const T *)a.k.p + b * a.k.sb + (h / a.k.group) * a.k.sh + dk0;
    const T *const vp = (const T *)a.v.p + b * a.v.sb + (h / a.v.group) * a.v.sh + dv0;
    const T *const qp = (const T *)a.q.p + b * a.q.sb + (h / a.q.group) * a.q.sh + dk0;
    const T *const op = (const T *)grad.p + b * grad.sb + (h / grad.group) * grad.sh + dv0;
    const int chunks = (int)((end - begin + C - 1) / C);
    int64_t r0 = end - (int64_t)chunks * C;
    const int row_base_of_lane = KTile::row_base(ln, half), v_row_base_of_lane = VTile::row_base(ln, half);
    int k_bases_of_lane[KTile::kColumnBases], v_bases_of_lane[VTile::kColumnBases];
    KTile::column_bases(k_bases_of_lane, lane);
    VTile::column_bases(v_bases_of_lane, lane);
    // (as in chunk_kernel)
    const bool grows = g2 > 0.f && chunks == 1;
    const int padded = grows ? (int)(begin - r0) : 0, most = C - padded;
    const float g_state = uniform(grows && piece == 0 && !a.first ? 0.f : g2);
    if (threadIdx.x < C)
        table_left[threadIdx.x / 4][threadIdx.x % 4] = (int)threadIdx.x < padded ? 0.f : exp2f(g2 * (float)(C - 1 - (int)threadIdx.x));
    if (wave < CT) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int gap = 32 * wave + ln - acc_row(r, half);
            table_gap[wave][r / 4][lane][r % 4] = gap > 0 && gap < most ? (float)gap / kGap * exp2f(g2 * (float)gap) : 0.f;
        }
    }
    if (NW == 1 && CT == 2) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int gap = 32 + ln - acc_row(r, half);
            table_gap[CT - 1][r / 4][lane][r % 4] = gap < most ? (float)gap / kGap * exp2f(g2 * (float)gap) : 0.f;
        }
    }
    Fetch<T, DK, C, THREADS> fk, fq;
    Fetch<T, DV, C, THREADS> fv, fo;
    // (where registers do not hold a whole chunk, the tensors pass through them one after the other)
    auto fetch = [&](int64_t at, int pad) {
        fk.load(kp + at * a.k.st, (int)a.k.st, a.Kp - dk0, pad);
        if (!kAhead) fk.store(lds_k);
        fq.load(qp + at * a.q.st, (int)a.q.st, a.Kp - dk0, pad);
        if (!kAhead) fq.store(lds_q);
        fv.load(vp + at * a.v.st, (int)a.v.st, a.Vp - dv0, pad);
        if (!kAhead) fv.store(lds_v);
        fo.load(op + at * grad.st, (int)grad.st, a.Vp - dv0, pad);
        if (!kAhead) fo.store(lds_o);
    };
    auto store = [&]() {
        fk.store(lds_k);
        fq.store(lds_q);
        fv.store(lds_v);
        fo.store(lds_o);
    };
    if (kAhead && chunks > 0) fetch(r0, (int)(begin - r0));
    double total = 0;  // of chunks; terms of a chunk are added in 32 bits
    for (int c = 0; c < chunks; ++c, r0 += C) {
        const int pad = (int)max(begin - r0, (int64_t)0);
        __syncthreads();
        // (tokens of padding are rows of zeros: their factor is kept from turning around)
        if (c < 2 && threadIdx.x < C)
            table_since[threadIdx.x / 4][threadIdx.x % 4] = exp2f(g_state * (float)max((int)threadIdx.x + 1 - pad, 0));
        if (kAhead)
            store();
        else
            fetch(r0, pad);
        __syncthreads();
        if (kAhead && c + 1 < chunks) fetch(r0 + C, 0);
        int row_base = row_base_of_lane, v_row_base = v_row_base_of_lane, k_bases[KTile::kColumnBases],
            v_bases[VTile::kColumnBases];
        asm volatile("" : "+v"(row_base), "+v"(v_row_base));
#pragma unroll
        for (int g = 0; g < KTile::kColumnBases; ++g) {
            k_bases[g] = k_bases_of_lane[g];
            v_bases[g] = v_bases_of_lane[g] ^ (wave * 32 * (int)sizeof(T));
            asm volatile("" : "+v"(k_bases[g]), "+v"(v_bases[g]));
        }
        v_row_base ^= wave * 32 * (int)sizeof(T);

        float chunk = 0.f;
        // inside the chunk; this wave's channels of do . v
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                f32x16 scores = {}, pulls = {};
#pragma unroll
                for (int kk = 0; kk < DK / 16; ++kk) {
                    scores = mma(KTile::row(lds_k, row_base, j, kk), KTile::row(lds_q, row_base, i, kk), scores);
                    if (kk % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    pulls = mma(VTile::row(lds_v, v_row_base, j, kk), VTile::row(lds_o, v_row_base, i, kk), pulls);
                float sum = 0.f;
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const f32x4 f = table_gap[i - j][r4][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = scores[4 * r4 + e] * pulls[4 * r4 + e];
                        // (selected, not multiplied by zero: a later token may be infinite)
                        sum += i > j || acc_row(4 * r4 + e, half) < ln ? f[e] * x : 0.f;
                    }
                }
                chunk += kGap * sum;
            }

        // through the states, some tiles of rows at a time
        constexpr int kBlock = DKT < 4 ? DKT : 2;
#pragma unroll
        for (int t0 = 0; t0 < DKT; t0 += kBlock) {
            f32x16 G[kBlock], G1[kBlock];
#pragma unroll
            for (int t = 0; t < kBlock; ++t) G[t] = G1[t] = f32x16{};
#pragma unroll
            for (int kk = 0; kk < 2 * CT; ++kk) {
                // (the power first, then its exponent: their product may overflow where that with a small element does not)
                f32x8 o = widened(VTile::column(lds_o, v_bases, 0, kk)), o1;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] *= table_since[4 * kk + 2 * (e / 4) + half][e % 4];
                    o1[e] = (float)(16 * kk + acc_row(e, half) + 1 - pad) * o[e];
                }
                Frag<T> x[TERMS], x1[TERMS];
                split<T>(o, x);
                split<T>(o1, x1);
#pragma unroll
                for (int t = 0; t < kBlock; ++t) {
                    const Frag<T> q = KTile::column(lds_q, k_bases, t0 + t, kk);
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) {
                        G[t] = mma(q, x[i], G[t]);
                        G1[t] = mma(q, x1[i], G1[t]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t < kBlock; ++t) chunk += sum16(D[t0 + t] * G[t] + S[t0 + t] * G1[t]);
        }
        total += chunk;

        const float count = (float)(C - pad), whole = exp2f(g_state * count);
#pragma unroll
        for (int t = 0; t < DKT; ++t) {
            D[t] = whole * (D[t] + count * S[t]);
            S[t] *= whole;
        }
#pragma unroll
        for (int kk = 0; kk < 2 * CT; ++kk) {
            f32x8 v = widened(VTile::column(lds_v, v_bases, 0, kk)), v1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] *= table_left[4 * kk + 2 * (e / 4) + half][e % 4];
                v1[e] = (float)(C - 1 - 16 * kk - acc_row(e, half)) * v[e];
            }
            Frag<T> x[TERMS], x1[TERMS];
            split<T>(v, x);
            split<T>(v1, x1);
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
                const Frag<T> k = KTile::column(lds_k, k_bases, t, kk);
#pragma unroll
                for (int i = 0; i < TERMS; ++i) {
                    S[t] = mma(k, x[i], S[t]);
                    D[t] = mma(k, x1[i], D[t]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    total *= a.out_scale;
    // the gradient of the state behind the piece; not where there is no token, whatever it is
    if (chunks > 0) {
        load_state<DKT, NW, false>(S, back, b, h, n, a.pieces - piece - a.run, g2, dk0, dv0, dv, half);
#pragma unroll
        for (int t = 0; t < DKT; ++t) total += sum16(D[t] * S[t]);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) total += __shfl_xor(total, m);
    if (lane == 0) meet[wave] = total;
    __syncthreads();
    if (threadIdx.x > 0) return;
    for (int w = 1; w < NW; ++w) total += meet[w];
    partial[(((int64_t)blockIdx.y * slices + slice) * a.B + b) * a.H + h] = (float)total;
}

template <typename T, int DKT, int NW, int CT, int TERMS>
void launch_sweep(const Sweep &a, dim3 grid, int slices, hipStream_t stream) {
    if (a.out_float && sizeof(T) == 2)
        chunk_kernel<T, float, DKT, NW, CT, TERMS, false><<<grid, 64 * NW, 0, stream>>>(a, slices);
    else
        chunk_kernel<T, T, DKT, NW, CT, TERMS, false><<<grid, 64 * NW, 0, stream>>>(a, slices);
}

// Sequences of up to 32 tokens take chunks of 32 where longer ones have 64, half of which would be padding (1024 x 20 tokens, 16 heads
// of 64, from a state to a state: 155 us, in chunks of 64 238; 2048 x 8 tokens in training 630 and 1238).
template <typename T, int DKT, int NW, int TERMS>
void launch_width(const Sweep &a, bool fold, hipStream_t stream) {
    constexpr int CT = chunk_tiles<T>(DKT, NW);
    const int slices = (int)ceil_div(a.Dv, 32 * NW);
    const dim3 grid((unsigned)(slices * a.H), (unsigned)(fold ? a.pieces - a.run : a.pieces / a.run), (unsigned)a.B);
    if (fold) return chunk_kernel<T, T, DKT, NW, CT, TERMS, true><<<grid, 64 * NW, 0, stream>>>(a, slices);
    if (CT > 1 && a.L <= 32) return launch_sweep<T, DKT, NW, 1, TERMS>(a, grid, slices, stream);
    launch_sweep<T, DKT, NW, CT, TERMS>(a, grid, slices, stream);
}

// A state that is handed out in 32 bits is summed from all bits of its terms.  For one that only answers, through a copy in two terms of
// the type of the products, two terms of bf16 are enough; one would be off by as much as the rounding of an answer is.
template <typename T, int DKT, int NW>
void launch_terms(const Sweep &a, bool fold, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (a.exact_state) return launch_width<T, DKT, NW, 3>(a, fold, stream);
        launch_width<T, DKT, NW, 2>(a, fold, stream);
    } else {
        launch_width<T, DKT, NW, 1>(a, fold, stream);
    }
}

template <typename T, int DKT, int NW>
void launch_decay_width(const Sweep &a, const Sweep &back, const View &grad, float *partial, hipStream_t stream) {
    const int slices = decay_slices(a);
    const dim3 grid((unsigned)(slices * a.H), (unsigned)(a.pieces / a.run), (unsigned)a.B), block(64 * NW);
    decay_kernel<T, DKT, NW><<<grid, block, 0, stream>>>(a, back, grad, partial, slices);
}

}  // namespace

template <typename T, int DKT>
void launch_chunks(const Sweep &a, bool fold, hipStream_t stream) {
    if (a.Dv <= 32) return launch_terms<T, DKT, 1>(a, fold, stream);
    if (a.Dv <= 64) return launch_terms<T, DKT, 2>(a, fold, stream);
    launch_terms<T, DKT, 4>(a, fold, stream);
}

template <typename T, int DKT>
void launch_decay(const Sweep &a, const Sweep &back, const View &grad_out, float *partial, hipStream_t stream) {
    if (a.Dv <= 32) return launch_decay_width<T, DKT, 1>(a, back, grad_out, partial, stream);
    if (a.Dv <= 64) return launch_decay_width<T, DKT, 2>(a, back, grad_out, partial, stream);
    launch_decay_width<T, DKT, 4>(a, back, grad_out, partial, stream);
}

template void launch_chunks<float, PSIG_KEY_TILES>(const Sweep &, bool, hipStream_t);
template void launch_chunks<bf16, PSIG_KEY_TILES>(const Sweep &, bool, hipStream_t);
#if PSIG_KEY_TILES <= 4  // (wider states are dealt to blocks by 128 rows)
template void launch_decay<float, PSIG_KEY_TILES>(const Sweep &, const Sweep &, const View &, float *, hipStream_t);
template void launch_decay<bf16, PSIG_KEY_TILES>(const Sweep &, const Sweep &, const View &, float *, hipStream_t);
#endif

}  // namespace seq
}  // namespace psig
