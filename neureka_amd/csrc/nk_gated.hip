// nk_gated_matmul, nk_gated_matmul_backward: the gated half of a feed-forward block.
//
//     gate = X Wg      up = X Wu      H = f(gate) up
//     with the error E of H:  dg = E up f'(gate)   du = E f(gate)   dX = dg Wg^T + du Wu^T   dWg = X^T dg   dWu = X^T du
//
// Every product is result(m, n) = sum over l of A(m, l) B(n, l).  Two switches say where an operand's neighbours along l lie (next to each
// other, or a row apart), which covers X, its transpose and weights of either layout without a copy.  Two products that share A
// (forward, weight gradients) are PAIRED: a tile holds the same columns of both, half each, so that A is staged once for both and
// f(gate) up is formed in the registers that hold the sums.  dX is one product over a contraction of two segments, (dg, Wg) and then
// (du, Wu).  What bounds them and what runs:
//   few_rows_kernel        up to 32 rows (64 with few weights): the weights' bytes; straight from memory into registers
//   split_product_kernel   f32: the 16-bit matrix cores, which take floats as sums of 16-bit numbers; tiles through LDS
//   product_kernel         f64: the f64 matrix cores; straight from memory into registers
//   product_join_kernel    adds parts of the contraction where tiles alone would not fill the chip
//   gated_errors_kernel    dg and du, once, for the three products of the backward pass
#include "nk_internal.h"
#include "nk_scalar.h"

namespace nk {

// ---- the activations ----------------------------------------------------------------------------------------------
// f as the library's activations compute it (nk_scalar.h)
template <typename T> __device__ __forceinline__ T gated_fun(int fun, T x) {
    switch (fun) {
        case NK_FUN_RELU: return x >= T(0) ? x : x * T(.01);
        case NK_FUN_SIG:  return sigmoid(x);
        case NK_FUN_SILU: return x * sigmoid(x);
        case NK_FUN_GELU: return x * gelu_sigmoid(x);
        case NK_FUN_TANH: return tanh_ref(x);
        default:          return x;
    }
}
// f and f'.  1 - s is taken as the logistic function of the negated argument, and sech^2 as 4 e / (1 + e)^2: nothing cancels for large arguments.
template <typename T> __device__ __forceinline__ void gated_fun_and_slope(int fun, T x, T& f, T& slope) {
    switch (fun) {
        case NK_FUN_RELU: slope = x >= T(0) ? T(1) : T(.01); f = x >= T(0) ? x : x * T(.01); return;
        case NK_FUN_SIG: { const T s = sigmoid(x), c = sigmoid(-x); f = s; slope = s * c; return; }
        case NK_FUN_SILU: { const T s = sigmoid(x), c = sigmoid(-x); f = x * s; slope = s + f * c; return; }
        case NK_FUN_GELU: { const T s = gelu_sigmoid(x), c = gelu_sigmoid(-x); f = x * s; slope = s + T(1.702) * f * c; return; }
        case NK_FUN_TANH: {
            const T e = Num<T>::exp(T(-2) * Num<T>::abs(x)), d = T(1) + e;
            f = tanh_ref(x); slope = T(4) * e / (d * d); return;
        }
        default: f = x; slope = T(1); return;
    }
}

// ---- the products ----------------------------------------------------------------------------------------------------
template <typename T>
struct Product {
    const T* A[2]; int64_t lda;         // unpaired: one per segment of the contraction
    const T* B[2]; int64_t ldb;         // unpaired: one per segment; paired: one per half of the tile
    int rows, cols, inner;              // of one product (cols: of one half; inner: of one segment)
    int segments;
    int tiles_m, tiles_n, steps_per_part;   // a part: that many steps of BK along the contraction
    int64_t part_stride;                // elements from one part's results to the next's
    int fun;
    const int *a_scale, *b_scale[2];    // binary exponents of the rows of A and of B (per half), or null: see split_product_kernel
    T* out[3];                          // GATED: H, gate, up; STORE: the product (both halves); SUM: their sum
};
enum { STORE = 0, GATED = 1, SUM = 2 };      // SUM: both halves added into one result

template <typename T> struct Quad;
template <> struct Quad<float> {        // register v of lane l: row 4 (l / 16) + v, column l % 16 of a 16 x 16 tile
    typedef float Acc __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Acc mma(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int lane, int v) { return 4 * (lane >> 4) + v; }
};
template <> struct Quad<double> {       // row 4 v + l / 16
    typedef double Acc __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ Acc mma(double a, double b, Acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int lane, int v) { return 4 * v + (lane >> 4); }
};

// The tile a block owns: consecutive block ids go round the 8 XCDs, each of which gets a contiguous run of tiles (bands of 8
// tile rows, walked column by column), so that the blocks that share an L2 share operands.
__device__ __forceinline__ unsigned place_of(unsigned block, unsigned blocks) {
    const unsigned each = blocks / 8, rest = blocks % 8, xcd = block % 8, at = block / 8;
    return xcd * each + (xcd < rest ? xcd : rest) + at;
}
__device__ __forceinline__ void own_tile(unsigned block, unsigned tiles, int tiles_m, int tiles_n, int& tm, int& tn) {
    const unsigned id = place_of(block, tiles);
    const unsigned band = 8 * (unsigned)tiles_n, b = id / band, in = id - b * band;
    const unsigned height = (unsigned)tiles_m - b * 8 < 8 ? (unsigned)tiles_m - b * 8 : 8;
    tm = (int)(b * 8 + in % height);
    tn = (int)(in / height);
}

// The f64 products: tiles of 64 x 64, the contraction shared by the block's 4 wavefronts, chunks of 8 l in turn.  Every wavefront holds the
// whole tile (4 x 4 fragments of 16 x 16) and nothing it reads is another's, so its operands go from memory straight into the
// registers of the matrix instructions: 32 instructions of 64 cycles to a chunk of 8 l, whose eight 16-byte loads went out a chunk
// before.  No barrier until the sums meet in LDS, where each wavefront takes a quarter of the tile.
// 2048^3 forward 59 TFLOP/s, 512 x 512 x 2048 50 (tiles staged in LDS for 4 wavefronts of 32 x 32: 52 and 41): there the matrix cores are
// busy three quarters of the time that a unit has work, the rest is the first requests, the sums and f.
//
// Quarter q of a wavefront takes l = 2 q, 2 q + 1 of a chunk.  Operands that lie along l: a lane's two values are one load.  Operands that
// lie across: a lane loads two neighbouring rows (columns) of one l, so fragments 2 h and 2 h + 1 hold rows 32 h + 2 r and 32 h + 2 r + 1.
template <bool ALONG>
struct Strip {                                              // 64 rows of A (columns of B); PAIRED: 32 of either of two matrices
    const double* at[4];                                    // ALONG: a row each; across: the first of two, at[h] (from l = 2 q on either way)
    // `first[h]`: the row at which 32 rows of the strip start; rows past the end are read as the last ones, which the store leaves out
    __device__ __forceinline__ void place(const double* const (&from)[2], const int (&first)[2], int count, int64_t ld, int lane) {
        const int c = lane & 15, q = lane >> 4;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if constexpr (ALONG) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = first[h] + e * 16 + c;
                    at[2 * h + e] = from[h] + (int64_t)(r < count ? r : count - 1) * ld + 2 * q;
                }
            } else at[h] = from[h] + pair_of(first[h] + 2 * c, count) + (int64_t)(2 * q) * ld;
        }
    }
    static __device__ __forceinline__ int pair_of(int r, int count) { return r + 2 <= count ? r : count - 2; }
    // the row of the strip's fragment f that index r of the fragment stands for, given the 32 rows' first; -1: none
    static __device__ __forceinline__ int row_of(int first, int f, int r, int count) {
        if constexpr (ALONG) { const int m = first + (f & 1) * 16 + r; return m < count ? m : -1; }
        const int own = first + 2 * r, m = pair_of(own, count) + (f & 1);
        return m >= own && m < count ? m : -1;
    }
    __device__ __forceinline__ void load(double (&v)[4][2], int64_t shift, int64_t ld, int l0) const {      // v[fragment][l]
        typedef double V __attribute__((ext_vector_type(2), aligned(8)));
        if constexpr (ALONG) {
#pragma unroll
            for (int f = 0; f < 4; f++) {
                const V x = *(const V*)(at[f] + shift + l0);
                v[f][0] = x[0]; v[f][1] = x[1];
            }
        } else
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const V x = *(const V*)(at[h] + shift + (int64_t)(l0 + s) * ld);
                    v[2 * h][s] = x[0]; v[2 * h + 1][s] = x[1];
                }
    }
    // the same where the contraction ends inside the chunk: zero from `inner` on
    __device__ __forceinline__ void load_rest(double (&v)[4][2], int64_t shift, int64_t ld, int l0, int inner, int lane) const {
        const int l = l0 + 2 * (lane >> 4);
#pragma unroll
        for (int f = 0; f < 4; f++)
#pragma unroll
            for (int s = 0; s < 2; s++)
                v[f][s] = l + s < inner ? (ALONG ? at[f][shift + l0 + s] : at[f >> 1][shift + (int64_t)(l0 + s) * ld + (f & 1)]) : 0.0;
    }
};

template <bool A_ALONG, bool B_ALONG, bool PAIRED, int EPI>
__global__ __launch_bounds__(256, 2) void product_kernel(const Product<double> g) {
    typedef Quad<double> Q;
    typedef Q::Acc Acc;
    constexpr int BM = 64, HALF = PAIRED ? 32 : 64, KC = 8, BK = 16;
    __shared__ Acc sums[2][3][4][64];                       // two rows of fragments at a time, three wavefronts' shares
    const unsigned tiles = (unsigned)(g.tiles_m * g.tiles_n), part = blockIdx.x / tiles;
    int tm, tn;
    own_tile(blockIdx.x - part * tiles, tiles, g.tiles_m, g.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * HALF;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int a_first[2] = {m0, m0 + 32}, b_first[2] = {n0, PAIRED ? n0 : n0 + 32};
    Strip<A_ALONG> a;
    Strip<B_ALONG> b;
    const double *const a_from[2] = {g.A[0], g.A[0]}, *const b_from[2] = {g.B[0], PAIRED ? g.B[1] : g.B[0]};
    a.place(a_from, a_first, g.rows, g.lda, lane);
    b.place(b_from, b_first, g.cols, g.ldb, lane);
    // whole steps of all segments first, g.steps_per_part of them per part; the last part also takes what is left of each segment
    const int whole = g.inner / BK, all = whole * g.segments;
    const int first = (int)part * g.steps_per_part < all ? (int)part * g.steps_per_part : all;
    const int last = first + g.steps_per_part < all ? first + g.steps_per_part : all;
    const int64_t a_shift = PAIRED ? 0 : g.A[1] - g.A[0], b_shift = PAIRED ? 0 : g.B[1] - g.B[0];       // to the second segment
    struct Chunk { double a[4][2], b[4][2]; };
    const int chunks = 2 * last;                            // (a wavefront takes every fourth: two that share the lines of what lies along l at a time)
    const auto request = [&](Chunk& k, int c) {             // past the end: the last one once more
        c = c < chunks ? c : chunks - 1;
        const bool second = !PAIRED && c >= 2 * whole;
        const int l0 = (second ? c - 2 * whole : c) * KC;
        a.load(k.a, second ? a_shift : 0, g.lda, l0);
        b.load(k.b, second ? b_shift : 0, g.ldb, l0);
    };
    Acc acc[4][4] = {};
    const auto multiply = [&](const Chunk& k) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = Q::mma(k.a[i][s], k.b[j][s], acc[i][j]);
    };
    if (2 * first + wave < chunks) {
        Chunk one, two;
        request(one, 2 * first + wave);
        int c = 2 * first + wave;
        for (; c + 4 < chunks; c += 8) {
            request(two, c + 4);
            __builtin_amdgcn_sched_barrier(0);               // the requests go out before the products of the chunk that is here
            multiply(one);
            request(one, c + 8);
            __builtin_amdgcn_sched_barrier(0);
            multiply(two);
        }
        if (c < chunks) multiply(one);
    }
    if (wave == 3 && g.inner % BK != 0 && last == all)
        for (int segment = 0; segment < g.segments; segment++)
            for (int l0 = whole * BK; l0 < g.inner; l0 += KC) {
                Chunk rest;
                a.load_rest(rest.a, segment ? a_shift : 0, g.lda, l0, g.inner, lane);
                b.load_rest(rest.b, segment ? b_shift : 0, g.ldb, l0, g.inner, lane);
                multiply(rest);
            }
    // row i of fragments belongs to wavefront i, which adds the shares of the others to its own in a fixed order
#pragma unroll
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int i = pass * 2 + e;
            if (wave != i)
#pragma unroll
                for (int j = 0; j < 4; j++) sums[e][wave - (wave > i)][j][lane] = acc[i][j];
        }
        __syncthreads();
        if (wave >> 1 == pass)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                Acc x = wave & 1 ? acc[pass * 2 + 1][j] : acc[pass * 2][j];
#pragma unroll
                for (int w = 0; w < 3; w++) x += sums[wave & 1][w][j][lane];
                acc[0][j] = x;                               // (its own share is not needed again, nor is row 0 of any other wavefront)
            }
        if (pass == 0) __syncthreads();
    }
    const int64_t shift = (int64_t)part * g.part_stride;
    const int c = lane & 15;
#pragma unroll
    for (int v = 0; v < 4; v++) {
        const int m = a.row_of(m0 + (wave >> 1) * 32, wave, Q::row(lane, v), g.rows);
        if (m < 0) continue;
        const int64_t row = (int64_t)m * g.cols + shift;
#pragma unroll
        for (int j = 0; j < (PAIRED ? 2 : 4); j++) {
            const int n = b.row_of(n0 + (j >> 1) * 32, j, c, g.cols);
            if (n < 0) continue;
            const double x = acc[0][j][v];
            if constexpr (!PAIRED) g.out[0][row + n] = x;
            else {
                const double y = acc[0][j + 2][v];
                if constexpr (EPI == GATED) {
                    g.out[0][row + n] = gated_fun(g.fun, x) * y;
                    if (g.out[1]) { g.out[1][row + n] = x; g.out[2][row + n] = y; }
                } else { g.out[0][row + n] = x; g.out[1][row + n] = y; }
            }
        }
    }
}

// ---- f32 products on the 16-bit matrix cores --------------------------------------------------------------------------
// The 16-bit instructions do 16 times the work of the f32 one per cycle and add exact partial products in f32, so a product of
// sums of 16-bit numbers costs less than the product of the floats they make up, and loses no more on ordinary operands.  Two ways (PLANES):
//
// 3: bfloat16, any operands.  A float is the sum of three, each the rest of the ones before rounded to nearest: 3 x 8 bits hold its 24
// (below 2^-110 the last leaves bfloat16's range: off by at most 2^-134).  The six largest of the nine partial products are added,
// x0 y0, x0 y1, x1 y0, x1 y1, x0 y2, x2 y0; the rest is at most 2^-25 of x y each.  A non-finite operand has no such sum
// (infinity - infinity), so a wavefront that finds a non-finite result computes that fragment of its tile once more with the f32
// instruction, straight from memory: what comes out is what f32 arithmetic gives.
//
// 2: half precision, half as many partial products: x0 y0, x0 y1, x1 y0.  Two halves hold a float to 2^-23 of it (2^-25 on average)
// and x1 y1 is at most 2^-22 of x y (2^-25 on average, of either sign), as long as they stay within the type's few binades.
// So a launch before finds, for every row of A and of B, the power of two that brings its largest magnitude to [2^14, 2^15).  The planes
// end at multiples of 2^-24, so a number is off by at most 2^-25 there: 2^-19 of itself or less from 2^-6 on, too much below.
// What such SMALL numbers are worth depends on what they meet (zeros may stand where their row is large), so no property of a row
// alone can tell.  The launch counts them, and each result is judged by what it came to: with a and b small numbers in its row and its column,
// each of which meets less than 2^15, it is off by less than (a + b) 2^-10 (1 + 2^-9), so one of UNCERTAIN (a + b) or more is right to 2^-18.
// A result below that is computed again from the floats.  In all, an error of at most 2^-17 of the sum of |x y|, with whatever rows meet; on
// average the planes' 2^-25.  Rows of which more than two and a 256th are small, where many results would have to be computed again, and
// rows with an infinity or NaN are marked, and a tile with a marked row takes three planes.  Of rows of 4096 normally distributed numbers one in 130
// has a small one, and one result in 10^9 is computed again; rows of dg (products of two such numbers and a slope) have one or two, eight at most.
constexpr int MARKED = 1 << 30, EMPTY = 1 << 29;             // notes on a row: three planes; nothing but zeros; else how many are small, and the exponent
constexpr int MOST_SMALL = (1 << 20) - 1;
constexpr float UNCERTAIN = 260.0f;                          // 2^-10 (1 + 2^-9) / 2^-18, rounded up
__device__ __forceinline__ int note_of(int exponent, int small) { return small << 9 | (exponent + 256); }
__device__ __forceinline__ int exponent_of(int note) { return (note & 511) - 256; }
__device__ __forceinline__ int small_of(int note) { return note >> 9 & MOST_SMALL; }
// the least magnitude, in the planes' scale, of a result that is certain; a row of zeros has results of zero whatever it meets
__device__ __forceinline__ float least_certain(int a, int b) { return (a | b) & EMPTY ? 0.0f : UNCERTAIN * (float)(small_of(a) + small_of(b)); }
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// two floats -> their three bfloat16 pairs
__device__ __forceinline__ void split_pair(float x, float y, unsigned (&p)[3]) {
#pragma unroll
    for (int k = 0; k < 3; k++) {
        const f32x2 v = {x, y};
        p[k] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
        if (k < 2) {
            x -= __builtin_bit_cast(float, p[k] << 16);
            y -= __builtin_bit_cast(float, p[k] & 0xffff0000u);
        }
    }
}
// two floats times a power of two (exact) -> their two pairs of halves; the rest is formed by a multiply-add that takes the half as it is
__device__ __forceinline__ void split_pair(float x, float y, float by, unsigned (&p)[2]) {
    const f16x2 high = __builtin_convertvector((f32x2{x * by, y * by}), f16x2);
    const f32x2 rest = {__builtin_fmaf(x, by, -(float)high[0]), __builtin_fmaf(y, by, -(float)high[1])};
    p[0] = __builtin_bit_cast(unsigned, high);
    p[1] = __builtin_bit_cast(unsigned, __builtin_convertvector(rest, f16x2));
}
template <int PLANES> struct Partial;
template <> struct Partial<3> {
    static constexpr int N = 6, A[N] = {0, 1, 2, 0, 1, 0}, B[N] = {0, 0, 0, 1, 1, 2};
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Partial<2> {
    static constexpr int N = 3, A[N] = {0, 1, 0}, B[N] = {0, 0, 1};
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// The notes on up to five operands' rows (`count` rows of `length`, together with those of a second matrix where there is
// one), blocks dealt out operand by operand.  Rows that lie along memory: a wavefront each, 64 stretches of every 64th 4 elements.
// Rows across memory: 32 of them per block, 64 stretches of every 64th element.  A stretch whose third least number is
// small for its row is read again to count.  Bound by memory: three operands of 4096 x 4096 in 53-60 us, 3.3-3.8 TB/s.
struct ScaleJob { const float* p[2]; int64_t ld; int count, length; bool along; int* out; unsigned blocks; };
struct ScaleJobs { ScaleJob job[5]; int n; };
__device__ __forceinline__ unsigned magnitude(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }
struct Range {                                               // of the magnitudes of a stretch, as their bits
    unsigned most = 0, least[3] = {~0u, ~0u, ~0u};          // the least other than zero, less one, in order
    __device__ __forceinline__ void add(float x) {
        const unsigned u = magnitude(x);
        most = u > most ? u : most;
        unsigned w = u - 1;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const unsigned above = w > least[k] ? w : least[k];
            least[k] = w < least[k] ? w : least[k];
            w = above;
        }
    }
    // how many are small, where the third is not
    __device__ __forceinline__ unsigned below(unsigned bound) const { return (least[0] < bound) + (least[1] < bound); }
};
// A magnitude other than zero is small in its row if, less one, it is below this: below 2^-6 times 2^14 over the largest's power of two.  (A largest
// number below 2^-111 is brought up by 2^126 alone: then even the least of the floats are multiples of 2^-23 there, and exact.)
__device__ __forceinline__ unsigned small_bound(unsigned largest) {
    const unsigned e = largest >> 23;
    return (e <= 15 || e >= 255 ? 1u : e <= 20 ? 1u << (e + 2) : (e - 20) << 23) - 1;
}
__device__ __forceinline__ int note_on(unsigned largest, unsigned small, int64_t elements) {
    const int64_t most = 2 + elements / 256;
    if (largest >= 0x7f800000u || small > (most < MOST_SMALL ? most : MOST_SMALL)) return MARKED;
    const int e = 14 + 127 - (int)(largest >> 23);
    return largest == 0 ? EMPTY | note_of(0, 0) : note_of(e < 126 ? e : 126, (int)small);
}

__global__ __launch_bounds__(512) void operand_scales_kernel(const ScaleJobs jobs) {
    unsigned block = blockIdx.x;
    int which = 0;
    while (which + 1 < jobs.n && block >= jobs.job[which].blocks) block -= jobs.job[which++].blocks;
    const ScaleJob j = jobs.job[which];
    const int64_t elements = (int64_t)j.length * (j.p[1] ? 2 : 1);
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    if (j.along) {
        const int row = (int)block * 8 + wave;
        if (row >= j.count) return;
        const auto visit = [&](auto take) {                  // the lane's stretch, of both matrices
            for (int k = 0; k < 2; k++) {
                if (!j.p[k]) continue;
                const float* const at = j.p[k] + (int64_t)row * j.ld;
                int i = lane * 4;
                for (; i + 3 * 256 + 4 <= j.length; i += 4 * 256) {          // four requests on their way
                    f32x4 v[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) v[u] = *(const f32x4_any*)(at + i + u * 256);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) take(v[u][e]);
                }
                for (; i + 4 <= j.length; i += 256) {
                    const f32x4 v = *(const f32x4_any*)(at + i);
#pragma unroll
                    for (int e = 0; e < 4; e++) take(v[e]);
                }
                for (; i < j.length; i++) take(at[i]);
            }
        };
        Range m;
        visit([&](float x) { m.add(x); });
        unsigned largest = m.most;
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) { const unsigned o = __shfl_xor(largest, step); largest = o > largest ? o : largest; }
        const unsigned bound = small_bound(largest);
        unsigned small = m.below(bound);
        if (m.least[2] < bound) small = 0, visit([&](float x) { small += magnitude(x) - 1 < bound; });
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) small += __shfl_xor(small, step);
        if (lane == 0) j.out[row] = note_on(largest, small, elements);
        return;
    }
    // lane: 4 neighbouring rows c .. c + 3 of the block's 32, stretch 8 wave + lane / 8
    __shared__ unsigned waves_largest[8][32], waves_small[8][32];
    const int q = lane & 7, c = (int)block * 32 + q * 4, first = wave * 8 + (lane >> 3);
    const auto visit = [&](auto take) {
        for (int k = 0; k < 2; k++) {
            if (!j.p[k]) continue;
            if (c + 4 <= j.count) {
                const float* const at = j.p[k] + c;
                int l = first;
                for (; l + 7 * 64 < j.length; l += 8 * 64) {                 // eight requests on their way
                    f32x4 v[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) v[u] = *(const f32x4_any*)(at + (int64_t)(l + u * 64) * j.ld);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int u = 0; u < 8; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) take(e, v[u][e]);
                }
                for (; l < j.length; l += 64) {
                    const f32x4 v = *(const f32x4_any*)(at + (int64_t)l * j.ld);
#pragma unroll
                    for (int e = 0; e < 4; e++) take(e, v[e]);
                }
            } else
                for (int l = first; l < j.length; l += 64)
#pragma unroll
                    for (int e = 0; e < 4; e++) if (c + e < j.count) take(e, j.p[k][(int64_t)l * j.ld + c + e]);
        }
    };
    Range m[4];
    visit([&](int e, float x) { m[e].add(x); });
    unsigned largest[4] = {m[0].most, m[1].most, m[2].most, m[3].most};
#pragma unroll
    for (int step = 8; step < 64; step <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) { const unsigned o = __shfl_xor(largest[e], step); largest[e] = o > largest[e] ? o : largest[e]; }
    if (lane < 8)
#pragma unroll
        for (int e = 0; e < 4; e++) waves_largest[wave][q * 4 + e] = largest[e];
    __syncthreads();
    unsigned bound[4], small[4];
    bool look = false;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        for (int w = 0; w < 8; w++) { const unsigned o = waves_largest[w][q * 4 + e]; largest[e] = o > largest[e] ? o : largest[e]; }
        bound[e] = small_bound(largest[e]);
        small[e] = m[e].below(bound[e]);
        look |= m[e].least[2] < bound[e];
    }
    if (look) {
#pragma unroll
        for (int e = 0; e < 4; e++) small[e] = 0;
        visit([&](int e, float x) { small[e] += magnitude(x) - 1 < bound[e]; });
    }
#pragma unroll
    for (int step = 8; step < 64; step <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) small[e] += __shfl_xor(small[e], step);
    if (lane < 8)
#pragma unroll
        for (int e = 0; e < 4; e++) waves_small[wave][q * 4 + e] = small[e];
    __syncthreads();
    if (wave == 0 && lane < 8)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            unsigned all = 0;
            for (int w = 0; w < 8; w++) all += waves_small[w][q * 4 + e];
            if (c + e < j.count) j.out[c + e] = note_on(largest[e], all, elements);
        }
}

__device__ __forceinline__ void lds_barrier() {             // orders LDS only: requests to memory stay in flight
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// LDS holds an operand's slice (WIDTH rows x 16 l) as PLANES planes of fragments of 32 rows x 16 l in the order in which the
// lanes of v_mfma_f32_32x32x16 take them: lane l gets the 8 values of row l % 32 from 8 (l / 32) on, 16 bytes.  The upper half's
// rows are rotated by 8 (row ^ 8) so that the writes below do not meet in one bank; a read is 1 KiB without a gap either way.
template <int PLANES, int WIDTH, bool ALONG, int THREADS>
struct SplitShare {
    static constexpr int E = WIDTH * 16 / THREADS;          // elements per thread: 4 or 8
    static constexpr unsigned PLANE = WIDTH * 32;           // bytes
    static_assert(E == 4 || E == 8, "a thread moves one or two times four elements");
    float v[2][E];                                          // two slices on their way
    const float* base[E / 4];                               // ALONG: the thread's rows; else: its column (base[0])
    float scale[E / 4];                                     // two planes: their powers of two
    int l_of;                                               // first l of the thread inside a slice

    __device__ __forceinline__ void place(const float* a, int64_t ld, int first, int count, int t, int half_of_columns, const float* other,
                                          const int* notes, const int* other_notes) {
        // half_of_columns > 0: rows from there on belong to the second matrix of a pair
#pragma unroll
        for (int u = 0; u < E / 4; u++) {
            int r = ALONG ? (t + u * THREADS) >> 2 : t % WIDTH;
            const float* from = a;
            const int* note = notes;
            if (half_of_columns > 0 && r >= half_of_columns) { r -= half_of_columns; from = other; note = other_notes; }
            const int64_t row = first + r < count ? first + r : count - 1;       // past the end: the last one, its results are not stored
            base[u] = from + row * (ALONG ? ld : 1);
            if constexpr (PLANES == 2) scale[u] = __builtin_bit_cast(float, (unsigned)(exponent_of(note[row]) + 127) << 23);
        }
        l_of = ALONG ? (t & 3) * 4 : __builtin_amdgcn_readfirstlane(t / WIDTH) * E;
    }
    // shift: from the first segment to this one.  WHOLE: all 16 l of the slice exist; else what lies past `inner` is zero.
    template <int SET, bool WHOLE>
    __device__ __forceinline__ void load(int64_t shift, int64_t ld, int l0, int inner) {
        const int l = l0 + l_of;
        if constexpr (ALONG) {
#pragma unroll
            for (int u = 0; u < E / 4; u++) {
                const float* const at = base[u] + shift + l;
                if constexpr (WHOLE) {
                    const f32x4 q = *(const f32x4_any*)at;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[SET][u * 4 + e] = q[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) v[SET][u * 4 + e] = l + e < inner ? at[e] : 0.0f;
                }
            }
        } else {
            const float* const at = base[0] + shift + (int64_t)l * ld;
#pragma unroll
            for (int e = 0; e < E; e++) v[SET][e] = WHOLE || l + e < inner ? at[(int64_t)e * ld] : 0.0f;
        }
    }
    template <int SET>
    __device__ __forceinline__ void store(unsigned char* lds, int t) const {
        unsigned p[E / 2][PLANES];
#pragma unroll
        for (int e = 0; e < E / 2; e++) {
            if constexpr (PLANES == 2) split_pair(v[SET][2 * e], v[SET][2 * e + 1], scale[ALONG ? e / 2 : 0], p[e]);
            else split_pair(v[SET][2 * e], v[SET][2 * e + 1], p[e]);
        }
        if constexpr (ALONG) {
            const int q = t & 3, high = q >> 1;
#pragma unroll
            for (int u = 0; u < E / 4; u++) {
                const int r = (t + u * THREADS) >> 2;
                unsigned char* const at = lds + (r >> 5) * 1024 + high * 512 + ((r & 31) ^ (high * 8)) * 16 + (q & 1) * 8;
#pragma unroll
                for (int k = 0; k < PLANES; k++) *(uint2*)(at + k * PLANE) = make_uint2(p[u * 2][k], p[u * 2 + 1][k]);
            }
        } else {
            const int r = t % WIDTH, l = l_of, high = l >> 3;
            unsigned char* const at = lds + (r >> 5) * 1024 + high * 512 + ((r & 31) ^ (high * 8)) * 16 + (l & 4) * 2;
#pragma unroll
            for (int k = 0; k < PLANES; k++) {
                if constexpr (E == 8) *(uint4*)(at + k * PLANE) = make_uint4(p[0][k], p[1][k], p[2][k], p[3][k]);
                else                  *(uint2*)(at + k * PLANE) = make_uint2(p[0][k], p[1][k]);
            }
        }
    }
};

// Three tile sizes: 256 x 256 (8 wavefronts of 128 x 64: 48 KiB of LDS reads for 48 matrix instructions of a slice), 256 x 128 and
// 128 x 128.  4096^3 forward, two planes: 740-755 us, 1.1e15 operations on halves a second, 364-372 TFLOP/s of float products (the f32
// instruction's peak is 157, a library's product of floats reaches 154).  The clock falls to 1.7 GHz under it with the matrix cores busy 61 %
// of the cycles, as under any dense product of 16-bit numbers here (a library's product of bfloat16, 8192^3: 1.3e15); without the
// requests to memory and the splitting the same loop takes 605 us.  Three planes: 1199 us.
//
// WM x WN wavefronts, each with a tile of FI x FJ fragments of 32 x 32.  PAIRED: the first half of a wavefront's column
// fragments comes from the first product, the second half from the second.
template <int PLANES, int WM, int WN, int FI, int FJ, bool A_ALONG, bool B_ALONG, bool PAIRED, int EPI>
__device__ __forceinline__ void split_product_tile(const Product<float>& g, unsigned char* lds, unsigned part, int m0, int n0) {
    constexpr int THREADS = WM * WN * 64, BM = WM * FI * 32, BN = WN * FJ * 32, HALF = PAIRED ? BN / 2 : BN;
    typedef SplitShare<PLANES, BM, A_ALONG, THREADS> AShare;
    typedef SplitShare<PLANES, BN, B_ALONG, THREADS> BShare;
    typedef Partial<PLANES> Part;
    constexpr unsigned A_BYTES = PLANES * AShare::PLANE, BUFFER = A_BYTES + PLANES * BShare::PLANE;
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, wm = wave / WN, wn = wave % WN;
    // the note on the tile's row r, column c (columns of a pair: the first product's, then the second's)
    const auto row_note = [&](int r) { return g.a_scale[m0 + r < g.rows ? m0 + r : g.rows - 1]; };
    const auto column_note = [&](int c) {
        const int n = n0 + (PAIRED && c >= HALF ? c - HALF : c);
        return g.b_scale[PAIRED && c >= HALF][n < g.cols ? n : g.cols - 1];
    };
    AShare a;
    BShare b;
    a.place(g.A[0], g.lda, m0, g.rows, t, 0, nullptr, g.a_scale, nullptr);
    b.place(g.B[0], g.ldb, n0, g.cols, t, PAIRED ? HALF : 0, g.B[1], g.b_scale[0], g.b_scale[1]);
    const int64_t a_shift = g.segments > 1 ? g.A[1] - g.A[0] : 0, b_shift = g.segments > 1 ? g.B[1] - g.B[0] : 0;
    // Whole slices of all segments first, g.steps_per_part of them per part; the last part also takes what is left of each segment.
    const int whole = g.inner / 16, all = whole * g.segments;
    const int first = (int)part * g.steps_per_part < all ? (int)part * g.steps_per_part : all;
    const int last = first + g.steps_per_part < all ? first + g.steps_per_part : all;
    const auto request_a = [&](auto set, int s) {
        const int segment = s >= whole;
        a.template load<decltype(set)::value, true>(segment ? a_shift : 0, g.lda, (s - segment * whole) * 16, g.inner);
    };
    const auto request_b = [&](auto set, int s) {
        const int segment = s >= whole;
        b.template load<decltype(set)::value, true>(segment ? b_shift : 0, g.ldb, (s - segment * whole) * 16, g.inner);
    };
    const auto column_block = [&](int j) { return PAIRED ? (j / (FJ / 2)) * (BN / 64) + wn * (FJ / 2) + j % (FJ / 2) : wn * FJ + j; };
    const unsigned mine = (unsigned)((lane >> 5) * 512 + (((lane & 31) ^ ((lane >> 5) * 8)) * 16));
    f32x16 acc[FI][FJ] = {};
    const auto read_a = [&](const unsigned char* from, int i, u32x4 (&f)[PLANES]) {
#pragma unroll
        for (int k = 0; k < PLANES; k++) f[k] = *(const u32x4*)(from + mine + k * AShare::PLANE + (wm * FI + i) * 1024);
    };
    const auto read_b = [&](const unsigned char* from, u32x4 (&f)[FJ][PLANES]) {
#pragma unroll
        for (int k = 0; k < PLANES; k++)
#pragma unroll
            for (int j = 0; j < FJ; j++) f[j][k] = *(const u32x4*)(from + mine + A_BYTES + k * BShare::PLANE + column_block(j) * 1024);
    };
    const auto multiply = [&](int i, const u32x4 (&af)[PLANES], const u32x4 (&bf)[FJ][PLANES]) {
#pragma unroll
        for (int c = 0; c < Part::N; c++)
#pragma unroll
            for (int j = 0; j < FJ; j++) acc[i][j] = Part::mma(af[Part::A[c]], bf[j][Part::B[c]], acc[i][j]);
    };

    if (first < last) {
        // A slice is one block without a branch.  Slice s is in LDS and the first fragments of it in registers; slices s + 1 and s + 2 are in
        // registers as floats or on their way (one slice takes 1.5 us, less than a loaded memory's answer: with slice s + 1 alone
        // on its way 4096^3 took 770 us).  s + 1 goes to LDS between the matrix instructions and its registers are asked for s + 3 (past
        // the end: the last slice once more).  The barrier stands before the last rows of fragments: behind it, while those are multiplied,
        // the first fragments of the next slice are read.
        typedef std::integral_constant<int, 0> Even;
        typedef std::integral_constant<int, 1> Odd;
        const auto clamp = [&](int s) { return s < last ? s : last - 1; };
        request_a(Even(), first); request_b(Even(), first);
        request_a(Odd(), clamp(first + 1)); request_b(Odd(), clamp(first + 1));
        a.template store<0>(lds, t); b.template store<0>(lds + A_BYTES, t);
        request_a(Even(), clamp(first + 2)); request_b(Even(), clamp(first + 2));
        lds_barrier();
        // rows of fragments multiplied before the barrier; the others' fragments wait in registers
        constexpr int BEFORE = PLANES == 2 ? FI / 2 : FI - 1, HELD = FI - BEFORE + 1;
        u32x4 bf[FJ][PLANES], af[HELD][PLANES];
        read_b(lds, bf);
        read_a(lds, 0, af[0]);
        const auto slice = [&](auto parity, int s) {
            constexpr int P = decltype(parity)::value;
            std::integral_constant<int, 1 - P> other;
            const unsigned char* const cur = lds + P * BUFFER;
            unsigned char* const next = lds + (1 - P) * BUFFER;
#pragma unroll
            for (int i = 0; i < BEFORE; i++) {
                if (i + 1 < BEFORE) read_a(cur, i + 1, af[(i + 1) % HELD]);
                else
#pragma unroll
                    for (int r = BEFORE; r < FI; r++) read_a(cur, r, af[r % HELD]);
                multiply(i, af[i % HELD], bf);
                if (i == 0) { a.template store<1 - P>(next, t); request_a(other, clamp(s + 3)); }
                if (i == (BEFORE > 1 ? 1 : 0)) { b.template store<1 - P>(next + A_BYTES, t); request_b(other, clamp(s + 3)); }
#pragma unroll
                for (int n = 0; n < Part::N * FJ; n++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);           // a matrix instruction,
                    __builtin_amdgcn_sched_group_barrier(0x002, PLANES == 2 ? 8 : 4, 0);           // vector arithmetic in its shadow,
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);           // an LDS read,
                    __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);           // an LDS write,
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);           // a request to memory
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            lds_barrier();
            u32x4 bn[FJ][PLANES], an[PLANES];
            read_a(next, 0, an);
            read_b(next, bn);
#pragma unroll
            for (int i = BEFORE; i < FI; i++) multiply(i, af[i % HELD], bf);
#pragma unroll
            for (int n = 0; n < PLANES * (1 + FJ); n++) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            // (without the empty statements the compiler moves these reads to the next slice, where nothing hides them)
#pragma unroll
            for (int k = 0; k < PLANES; k++) {
                asm volatile("" : "+v"(an[k]));
                af[0][k] = an[k];
#pragma unroll
                for (int j = 0; j < FJ; j++) {
                    asm volatile("" : "+v"(bn[j][k]));
                    bf[j][k] = bn[j][k];
                }
            }
        };
        int s = first;
        for (; s + 1 < last; s += 2) {
            slice(Even(), s);
            slice(Odd(), s + 1);
        }
        if (s < last) slice(Even(), s);
        lds_barrier();
    }
    if (g.inner % 16 != 0 && last == all) {
        for (int segment = 0; segment < g.segments; segment++) {
            a.template load<0, false>(segment ? a_shift : 0, g.lda, whole * 16, g.inner);
            b.template load<0, false>(segment ? b_shift : 0, g.ldb, whole * 16, g.inner);
            a.template store<0>(lds, t); b.template store<0>(lds + A_BYTES, t);
            lds_barrier();
            u32x4 bf[FJ][PLANES], af[PLANES];
            read_b(lds, bf);
#pragma unroll
            for (int i = 0; i < FI; i++) { read_a(lds, i, af); multiply(i, af, bf); }
            lds_barrier();
        }
    }

    // (two planes: the slices' memory takes the notes on the tile's rows and columns; every row in it is finite, and so is every sum)
    int* const notes = (int*)lds;
    if constexpr (PLANES == 2) {
        for (int r = t; r < BM; r += THREADS) notes[r] = row_note(r);
        for (int c = t; c < BN; c += THREADS) notes[BM + c] = column_note(c);
        lds_barrier();
    }
    // Register v of lane l: row 8 (v / 4) + 4 (l / 32) + v % 4, column l % 32 of a fragment.  Rows are counted from the tile's first, columns from
    // that of one product's half.
    const auto row_of = [&](int i, int v) { return (wm * FI + i) * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3); };
    const auto columns_of = [&](int j) { return (PAIRED ? wn * (FJ / 2) + j : wn * FJ + j) * 32; };
    const int64_t shift = (int64_t)part * g.part_stride;
    const auto put = [&](int r, int c, float x, float y) {
        const int m = m0 + r, n = n0 + c;
        if (m >= g.rows || n >= g.cols) return;
        const int64_t at = (int64_t)m * g.cols + n + shift;
        if constexpr (PAIRED && EPI == GATED) {
            g.out[0][at] = gated_fun(g.fun, x) * y;
            if (g.out[1]) { g.out[1][at] = x; g.out[2][at] = y; }
        } else {
            g.out[0][at] = x;
            if constexpr (PAIRED) g.out[1][at] = y;
        }
    };
    constexpr int SHOWN = PAIRED ? FJ / 2 : FJ;             // fragments per row of the wavefront's tile, of one product
    unsigned again = 0;                                     // fragments with results to be computed again
    unsigned* const open = (unsigned*)lds + BM + BN + wave * (FI * SHOWN * 64) + lane;        // two planes: which of the lane's, 64 words a fragment
    static_assert((BM + BN + WM * WN * FI * SHOWN * 64) * 4 <= 2 * BUFFER, "notes and results to be computed again fit where the slices were");
#pragma unroll
    for (int i = 0; i < FI; i++) {
        int most_small = 0;                                 // of the lane's rows
        if constexpr (PLANES == 2)
#pragma unroll
            for (int v = 0; v < 16; v++) { const int n = small_of(notes[row_of(i, v)]); most_small = n > most_small ? n : most_small; }
#pragma unroll
        for (int j = 0; j < SHOWN; j++) {
            const f32x16 &x = acc[i][j], &y = acc[i][PAIRED ? FJ / 2 + j : j];
            const int c = columns_of(j) + (lane & 31);
            if constexpr (PLANES == 3) {
                bool odd = false;
#pragma unroll
                for (int v = 0; v < 16; v++) odd |= !(__builtin_fabsf(x[v]) < INFINITY) || !(__builtin_fabsf(y[v]) < INFINITY);
                if (__any(odd)) { again |= 1u << (i * SHOWN + j); continue; }
#pragma unroll
                for (int v = 0; v < 16; v++) put(row_of(i, v), c, x[v], y[v]);
            } else {
                const int x_note = notes[BM + c], y_note = PAIRED ? notes[BM + HALF + c] : x_note;
                float least = INFINITY;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    least = __builtin_fminf(least, __builtin_fabsf(x[v]));
                    if constexpr (PAIRED) least = __builtin_fminf(least, __builtin_fabsf(y[v]));
                }
                const int small = small_of(x_note) > small_of(y_note) ? small_of(x_note) : small_of(y_note);
                unsigned uncertain = 0;
                if (__any(least < UNCERTAIN * (float)(most_small + small))) {
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const int note = notes[row_of(i, v)];
                        const bool bad = __builtin_fabsf(x[v]) < least_certain(note, x_note) || (PAIRED && __builtin_fabsf(y[v]) < least_certain(note, y_note));
                        uncertain |= (unsigned)(bad && m0 + row_of(i, v) < g.rows && n0 + c < g.cols) << v;
                    }
                    if (__any(uncertain != 0)) { again |= 1u << (i * SHOWN + j); open[(i * SHOWN + j) * 64] = uncertain; }
                }
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int r = row_of(i, v), e = exponent_of(notes[r]);
                    if (!(uncertain >> v & 1)) put(r, c, __builtin_ldexpf(x[v], -(e + exponent_of(x_note))), PAIRED ? __builtin_ldexpf(y[v], -(e + exponent_of(y_note))) : 0.0f);
                }
            }
        }
    }
    // What has to be computed again, from the floats as they are.  A slice of the part's whole ones, then what is left of each segment:
    const int turns = last - first + (last == all && g.inner % 16 != 0 ? g.segments : 0);
    const auto slice_of = [&](int turn, int& segment) {      // its first l
        const int s = first + turn, left = s - all;
        segment = left >= 0 ? left : s >= whole;
        return (left >= 0 ? whole : s - segment * whole) * 16;
    };
#pragma unroll 1
    for (int f = 0; f < FI * SHOWN; f++) {
        if (!(again >> f & 1)) continue;
        const int i = f / SHOWN, j = f % SHOWN;
        if constexpr (PLANES == 2) {
            // Up to 8 results: one after the other, by all lanes together (a fragment takes the time of about ten).
            unsigned mine = open[f * 64], count = __builtin_popcount(mine);
#pragma unroll
            for (int step = 32; step > 0; step >>= 1) count += __shfl_xor(count, step);
            if (count <= 8) {
                while (const uint64_t lanes = __ballot(mine != 0)) {
                    const int owner = __builtin_ctzll(lanes), v = __builtin_ctz(__shfl(mine, owner));
                    if (lane == owner) mine &= mine - 1;
                    const int r = (wm * FI + i) * 32 + 8 * (v >> 2) + 4 * (owner >> 5) + (v & 3), c = columns_of(j) + (owner & 31);
                    const int64_t am = (int64_t)(m0 + r) * (A_ALONG ? g.lda : 1), bn = (int64_t)(n0 + c) * (B_ALONG ? g.ldb : 1);
                    float x = 0, y = 0;
                    const auto add = [&](int segment, int from, int end) {
                        const float *const ap = g.A[segment] + am, *const bp = g.B[PAIRED ? 0 : segment] + bn, *const cp = g.B[1] + bn;
                        const int64_t a_step = A_ALONG ? 1 : g.lda, b_step = B_ALONG ? 1 : g.ldb;
                        int l = from + lane;
                        for (; l + 15 * 64 < end; l += 16 * 64) {            // 16 at a time on their way
                            float av[16], bv[16], cv[16];
#pragma unroll
                            for (int u = 0; u < 16; u++) {
                                av[u] = ap[(l + u * 64) * a_step];
                                bv[u] = bp[(l + u * 64) * b_step];
                                if constexpr (PAIRED) cv[u] = cp[(l + u * 64) * b_step];
                            }
#pragma unroll
                            for (int u = 0; u < 16; u++) {
                                x = __builtin_fmaf(av[u], bv[u], x);
                                if constexpr (PAIRED) y = __builtin_fmaf(av[u], cv[u], y);
                            }
                        }
                        for (; l < end; l += 64) {
                            const float av = ap[l * a_step];
                            x = __builtin_fmaf(av, bp[l * b_step], x);
                            if constexpr (PAIRED) y = __builtin_fmaf(av, cp[l * b_step], y);
                        }
                    };
                    for (int segment = 0; segment < g.segments; segment++) {
                        const int from = first - segment * whole, end = last - segment * whole;
                        add(segment, (from > 0 ? from : 0) * 16, (end < whole ? end : whole) * 16);
                        if (last == all) add(segment, whole * 16, g.inner);
                    }
#pragma unroll
                    for (int step = 32; step > 0; step >>= 1) { x += __shfl_xor(x, step); y += __shfl_xor(y, step); }
                    if (lane == 0) put(r, c, x, y);
                }
                continue;
            }
        }
        const int c = columns_of(j) + (lane & 31), m = m0 + (wm * FI + i) * 32 + (lane & 31), n = n0 + c;
        const int64_t am = (int64_t)(m < g.rows ? m : g.rows - 1) * (A_ALONG ? g.lda : 1), bn = (int64_t)(n < g.cols ? n : g.cols - 1) * (B_ALONG ? g.ldb : 1);
        f32x16 x = {}, y = {};
        struct Slice { float a[8], b[8], c[8]; };
        const auto request = [&](Slice& k, int turn) {
            int segment;
            const int l0 = slice_of(turn, segment);
            const float *const ap = g.A[segment] + am, *const bp = g.B[PAIRED ? 0 : segment] + bn, *const cp = g.B[1] + bn;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int l = l0 + 2 * e + (lane >> 5);
                const bool in = l < g.inner;
                const int64_t ao = (int64_t)(in ? l : 0) * (A_ALONG ? 1 : g.lda), bo = (int64_t)(in ? l : 0) * (B_ALONG ? 1 : g.ldb);
                const float av = ap[ao], bv = bp[bo];
                k.a[e] = in ? av : 0.0f;
                k.b[e] = in ? bv : 0.0f;
                if constexpr (PAIRED) { const float cv = cp[bo]; k.c[e] = in ? cv : 0.0f; }
            }
        };
        const auto multiply_floats = [&](const Slice& k) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x = __builtin_amdgcn_mfma_f32_32x32x2f32(k.a[e], k.b[e], x, 0, 0, 0);
                if constexpr (PAIRED) y = __builtin_amdgcn_mfma_f32_32x32x2f32(k.a[e], k.c[e], y, 0, 0, 0);
            }
        };
        Slice one, two;                                      // a slice on its way while the other is multiplied; past the end: the last once more
        request(one, 0);
        for (int turn = 0; turn < turns; turn += 2) {
            request(two, turn + 1 < turns ? turn + 1 : turns - 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply_floats(one);
            request(one, turn + 2 < turns ? turn + 2 : turns - 1);
            __builtin_amdgcn_sched_barrier(0);
            if (turn + 1 < turns) multiply_floats(two);
        }
#pragma unroll
        for (int v = 0; v < 16; v++) put(row_of(i, v), c, x[v], y[v]);
    }
}

// SCALED: two planes, or three where the tile holds a marked row.
template <bool SCALED, int WM, int WN, int FI, int FJ, bool A_ALONG, bool B_ALONG, bool PAIRED, int EPI>
__global__ __launch_bounds__(WM * WN * 64) void split_product_kernel(const Product<float> g) {
    constexpr int THREADS = WM * WN * 64, BM = WM * FI * 32, BN = WN * FJ * 32, HALF = PAIRED ? BN / 2 : BN;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];          // two buffers of both operands' planes
    const unsigned tiles = (unsigned)(g.tiles_m * g.tiles_n), part = blockIdx.x / tiles;
    int tm, tn;
    own_tile(blockIdx.x - part * tiles, tiles, g.tiles_m, g.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * HALF;
    if constexpr (SCALED) {
        bool marked = false;
        for (int r = threadIdx.x; r < BM; r += THREADS) marked |= g.a_scale[m0 + r < g.rows ? m0 + r : g.rows - 1] == MARKED;
        for (int c = threadIdx.x; c < BN; c += THREADS) {
            const int n = n0 + (c >= HALF ? c - HALF : c);
            marked |= g.b_scale[c >= HALF][n < g.cols ? n : g.cols - 1] == MARKED;
        }
        if (__syncthreads_or(marked) == 0) {
            split_product_tile<2, WM, WN, FI, FJ, A_ALONG, B_ALONG, PAIRED, EPI>(g, lds, part, m0, n0);
            return;
        }
    }
    split_product_tile<3, WM, WN, FI, FJ, A_ALONG, B_ALONG, PAIRED, EPI>(g, lds, part, m0, n0);
}

// ---- few rows ----------------------------------------------------------------------------------------------------------
// Up to 64 rows the weights' bytes bound the products, so they go from memory straight into the registers of the matrix
// instructions (16 x 16 x 4, of the element type itself), each element once.  A wavefront owns 16 CW columns of both products and
// RT x 16 rows; the block's wavefronts share the contraction, U chunks of KC at a time in turn, and add their sums through LDS
// in order.  Inside a chunk quarter q of a wavefront takes l from V q on, so that a lane's V values of A (and of weights stored
// along l) are one 16-byte load.
//
// What the memory delivers depends on how the requests lie (weights that no cache holds):
//  - Weights by row, in floats: one row tile reads 128 bytes of a row per wavefront (CW 2; 1 x 4096 x 4096 28 us, 64 bytes 34).  Two row
//    tiles and more read 64 and one chunk at a time (32 x 2048 x 3500 28 us, 128 bytes 35; four row tiles were measured this way alone).
//  - Weights stored along l: 128 bytes per column (U 2; 16 x 4096 x 4096 26 us, U 1 31); four row tiles take one chunk (64 x 2048 x
//    2048 19 us, U 2 24).  There every group starts at another place of the contraction, because groups that walk in step meet in the
//    same memory channels (33 us in step, 28 apart).
//  - Neighbouring columns belong to neighbouring blocks of one die, whose L2 holds the lines that they share where rows do not start with
//    a line (16 x 3001 x 1301 22 -> 18 us).
//  - Where the columns make fewer blocks than there are units, g.parts blocks share a group of columns: each adds its sums to memory,
//    and the one that arrives last adds them all, part by part.  As many parts as units hold at once, since a unit with two blocks
//    would end last (1 x 2048 x 3500, 110 groups: 2 parts 16 us, 3 parts 23).
//
// The shared sums are written and read by atomic accesses of the whole device, which pass the caches of the eight dies one
// by one; fences would write back and drop those caches whole (84 us instead of 27 for the call above).  What orders them: a wavefront
// waits for its stores before the block's barrier, behind which one thread announces the block's arrival.
template <typename Acc, typename T>
__device__ __forceinline__ void put_shared(T* at, const Acc& x) {
#pragma unroll
    for (int v = 0; v < 4; v++) __hip_atomic_store(at + v, x[v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename Acc, typename T>
__device__ __forceinline__ Acc get_shared(const T* at) {
    Acc x;
#pragma unroll
    for (int v = 0; v < 4; v++) x[v] = __hip_atomic_load(at + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return x;
}
template <typename T, int RT, int CW, bool ALONG, int EPI>
__global__ __launch_bounds__(512) void few_rows_kernel(const Product<T> g, int parts, T* partial, unsigned* arrived) {
    typedef Quad<T> Q;
    typedef typename Q::Acc Acc;
    constexpr int WAVES = 8, V = 16 / sizeof(T), KC = 4 * V, U = RT <= 2 && (ALONG || CW == 2) ? 2 : 1, NA = EPI == GATED ? 1 : 2, FRAGMENTS = RT * CW;
    typedef T VecV __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    typedef T VecC __attribute__((ext_vector_type(CW), aligned(sizeof(T))));
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, c = lane & 15, q = lane >> 4;
    const unsigned place = place_of(blockIdx.x, gridDim.x);
    const int part = place / (unsigned)g.tiles_n, group = place - (unsigned)part * (unsigned)g.tiles_n;
    // the lane's CW neighbouring columns (moved back where they would pass the last one; what it shares with others it does not store)
    const int own = group * 16 * CW + c * CW, n0 = own + CW <= g.cols ? own : g.cols - CW;
    const T *brow[2], *arow[NA][RT];
#pragma unroll
    for (int p = 0; p < 2; p++) brow[p] = g.B[p] + (int64_t)n0 * (ALONG ? g.ldb : 1);
#pragma unroll
    for (int p = 0; p < NA; p++)
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int m = r * 16 + c;
            arow[p][r] = g.A[p] + (int64_t)(m < g.rows ? m : g.rows - 1) * g.lda;
        }
    Acc acc[2][RT][CW] = {};
    struct Chunk { T a[NA][RT][V], b[2][CW][V]; };
    const auto load = [&](Chunk& k, int64_t l0) {            // a chunk that exists whole: no branch, so that the requests of several overlap
        const int64_t l = l0 + q * V;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            if constexpr (ALONG) {
#pragma unroll
                for (int j = 0; j < CW; j++) {
                    const VecV w = *(const VecV*)(brow[p] + j * g.ldb + l);
#pragma unroll
                    for (int s = 0; s < V; s++) k.b[p][j][s] = w[s];
                }
            } else
#pragma unroll
                for (int s = 0; s < V; s++) {
                    const VecC w = *(const VecC*)(brow[p] + (l + s) * g.ldb);
#pragma unroll
                    for (int j = 0; j < CW; j++) k.b[p][j][s] = w[j];
                }
        }
#pragma unroll
        for (int p = 0; p < NA; p++)
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const VecV x = *(const VecV*)(arow[p][r] + l);
#pragma unroll
                for (int s = 0; s < V; s++) k.a[p][r][s] = x[s];
            }
    };
    const auto load_rest = [&](Chunk& k, int64_t l0) {       // the last one, zeros past the end
        const int64_t l = l0 + q * V;
#pragma unroll
        for (int s = 0; s < V; s++) {
            const bool in = l + s < g.inner;
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int j = 0; j < CW; j++) k.b[p][j][s] = in ? brow[p][ALONG ? j * g.ldb + l + s : (l + s) * g.ldb + j] : T(0);
#pragma unroll
            for (int p = 0; p < NA; p++)
#pragma unroll
                for (int r = 0; r < RT; r++) k.a[p][r][s] = in ? arow[p][r][l + s] : T(0);
        }
    };
    const auto multiply = [&](const Chunk& k) {
#pragma unroll
        for (int s = 0; s < V; s++)
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int j = 0; j < CW; j++) acc[p][r][j] = Q::mma(k.a[NA == 1 ? 0 : p][r][s], k.b[p][j][s], acc[p][r][j]);
    };
    // The part's whole chunks, U at a time: wavefront w takes units w, w + WAVES, ...  What is left of the part, and the contraction's
    // last, partial chunk, belong to the last wavefront.
    const int whole = g.inner / KC, first = part * g.steps_per_part < whole ? part * g.steps_per_part : whole;
    const int last = first + g.steps_per_part < whole ? first + g.steps_per_part : whole;
    const int units = (last - first) / U, mine = units > wave ? (units - wave + WAVES - 1) / WAVES : 0;
    const int turn = ALONG && units > 0 ? (int)((unsigned)group * 17u % (unsigned)units) : 0;
    const auto at = [&](int i) {
        int unit = wave + i * WAVES + turn;
        if (ALONG) unit -= unit >= units ? units : 0;
        return (int64_t)(first + unit * U) * KC;
    };
    if (mine > 0) {
        Chunk now[U], next[U];
#pragma unroll
        for (int u = 0; u < U; u++) load(now[u], at(0) + u * KC);
        for (int i = 1; i < mine; i++) {
#pragma unroll
            for (int u = 0; u < U; u++) load(next[u], at(i) + u * KC);
            __builtin_amdgcn_sched_barrier(0);               // the requests go out before the products of the chunks that are here
#pragma unroll
            for (int u = 0; u < U; u++) multiply(now[u]);
#pragma unroll
            for (int u = 0; u < U; u++) now[u] = next[u];
        }
#pragma unroll
        for (int u = 0; u < U; u++) multiply(now[u]);
    }
    if (wave == WAVES - 1) {
        Chunk one;
        for (int k = first + units * U; k < last; k++) { load(one, (int64_t)k * KC); multiply(one); }
        if (last == whole && part == parts - 1 && g.inner % KC != 0) { load_rest(one, (int64_t)whole * KC); multiply(one); }
    }

    // the wavefronts' sums: [wave][product][row tile][column fragment][lane], a fragment's four values at a time
    Acc* const sums = (Acc*)lds;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int j = 0; j < CW; j++) sums[((wave * 2 + p) * FRAGMENTS + r * CW + j) * 64 + lane] = acc[p][r][j];
    __syncthreads();
    const auto total = [&](int f, int p) {
        Acc x = sums[(p * FRAGMENTS + f) * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; w++) x += sums[((w * 2 + p) * FRAGMENTS + f) * 64 + lane];
        return x;
    };
    T* const shared = partial + ((int64_t)group * (2 * FRAGMENTS * 64) + lane) * 4;          // part after part a whole result apart
    const int64_t apart = (int64_t)g.tiles_n * (2 * FRAGMENTS * 64) * 4;
    if (parts > 1) {
        for (int f = wave; f < 2 * FRAGMENTS; f += WAVES) put_shared(shared + part * apart + f * 256, total(f % FRAGMENTS, f / FRAGMENTS));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // this wavefront's sums have arrived
        __syncthreads();
        unsigned* const order = (unsigned*)lds;
        if (t == 0) {
            const unsigned n = __hip_atomic_fetch_add(arrived + group, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (n == (unsigned)parts - 1) __hip_atomic_store(arrived + group, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *order = n;
        }
        __syncthreads();
        if (*order != (unsigned)parts - 1) return;
    }
    for (int f = wave; f < FRAGMENTS; f += WAVES) {
        Acc x, y;
        if (parts > 1) {
            x = get_shared<Acc>(shared + f * 256);
            y = get_shared<Acc>(shared + (FRAGMENTS + f) * 256);
            for (int k = 1; k < parts; k++) {
                x += get_shared<Acc>(shared + k * apart + f * 256);
                y += get_shared<Acc>(shared + k * apart + (FRAGMENTS + f) * 256);
            }
        } else { x = total(f, 0); y = total(f, 1); }
        const int r = f / CW, n = n0 + f % CW;
        if (n < own || n >= g.cols) continue;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int m = r * 16 + Q::row(lane, v);
            if (m >= g.rows) continue;
            const int64_t o = (int64_t)m * g.cols + n;
            if constexpr (EPI == GATED) {
                g.out[0][o] = gated_fun(g.fun, x[v]) * y[v];
                if (g.out[1]) { g.out[1][o] = x[v]; g.out[2][o] = y[v]; }
            } else g.out[0][o] = x[v] + y[v];
        }
    }
}

// ---- parts of the contraction, added in order -----------------------------------------------------------------------
// partial: [parts][halves][n]; halves 2: the pair of products.  Four elements a thread; bound by memory (4 parts of 2048 x 1024
// floats 8 us, 5 TB/s).
template <typename T, bool PAIRED, int EPI>
__global__ __launch_bounds__(256) void product_join_kernel(const T* __restrict__ partial, int parts, int64_t n, int fun, T* out0, T* out1, T* out2) {
    typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    constexpr int HALVES = PAIRED ? 2 : 1;
    const auto finish = [&](int64_t at, T x, T y) {
        if constexpr (EPI == GATED) {
            out0[at] = gated_fun(fun, x) * y;
            if (out1) { out1[at] = x; out2[at] = y; }
        } else {
            out0[at] = x;
            if (PAIRED) out1[at] = y;
        }
    };
    if (i + 4 <= n) {
        V x = *(const V*)(partial + i), y = x;
        if (PAIRED) y = *(const V*)(partial + n + i);
#pragma unroll 4
        for (int p = 1; p < parts; p++) {
            x += *(const V*)(partial + (int64_t)p * HALVES * n + i);
            if (PAIRED) y += *(const V*)(partial + ((int64_t)p * HALVES + 1) * n + i);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) finish(i + e, x[e], y[e]);
        return;
    }
    for (int64_t at = i; at < n; at++) {
        T x = partial[at], y = PAIRED ? partial[n + at] : T(0);
        for (int p = 1; p < parts; p++) {
            x += partial[(int64_t)p * HALVES * n + at];
            if (PAIRED) y += partial[((int64_t)p * HALVES + 1) * n + at];
        }
        finish(at, x, y);
    }
}

// dg = E up f'(gate), du = E f(gate): five numbers through memory per element, four elements a thread (4096 x 4096 floats 57 us, 5.9 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void gated_errors_kernel(int fun, int64_t n, const T* __restrict__ error, const T* __restrict__ gate, const T* __restrict__ up,
                                                           T* __restrict__ d_gate, T* __restrict__ d_up) {
    typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    T f, slope;
    if (i + 4 <= n) {
        const V e = *(const V*)(error + i), g = *(const V*)(gate + i), u = *(const V*)(up + i);
        V dg, du;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            gated_fun_and_slope(fun, g[k], f, slope);
            dg[k] = e[k] * u[k] * slope;
            du[k] = e[k] * f;
        }
        *(V*)(d_gate + i) = dg;
        *(V*)(d_up + i) = du;
    } else
        for (int64_t at = i; at < n; at++) {
            gated_fun_and_slope(fun, gate[at], f, slope);
            d_gate[at] = error[at] * up[at] * slope;
            d_up[at] = error[at] * f;
        }
}

// ---- plans ---------------------------------------------------------------------------------------------------------------
struct Split { int edge_m, edge_n, tiles_m, tiles_n, parts, steps_per_part; };
// What a slice of 16 l takes in the kernels of one tile size, in microseconds, and the blocks of it that a unit runs at a time (two planes;
// with three every entry is near twice as long, which changes no choice): from 2048 x 1024 x 4096 and 4096^3, whole rounds; f64 512 x 512 x 2048.
struct TileCost { int edge_m, edge_n, per_unit; double slice_us; };
template <typename T> constexpr TileCost TILE_COSTS[] = {{256, 256, 1, 1.6}, {256, 128, 1, 0.92}, {128, 128, 2, 1.05}};
template <> constexpr TileCost TILE_COSTS<double>[] = {{64, 64, 2, 1.1}};

// The tile size and the number of parts of the contraction with the shortest estimate: rounds of blocks times slices, plus, with parts, a
// launch that reads them all and writes the sum.
template <typename T>
static Split plan(const Device* dev, bool paired, int64_t rows, int64_t cols, int64_t inner, int segments) {
    const int64_t cus = dev->props.multiProcessorCount, steps = inner / 16 * segments;      // whole slices
    Split best{};
    double best_us = 0;
    for (const TileCost& c : TILE_COSTS<T>) {
        Split s{};
        s.edge_m = c.edge_m; s.edge_n = c.edge_n;
        s.tiles_m = (int)((rows + c.edge_m - 1) / c.edge_m);
        s.tiles_n = (int)(paired ? (cols + c.edge_n / 2 - 1) / (c.edge_n / 2) : (cols + c.edge_n - 1) / c.edge_n);
        const int64_t tiles = (int64_t)s.tiles_m * s.tiles_n, slots = c.per_unit * cus;
        for (int64_t parts = 1; parts <= 16 && (parts == 1 || (steps / parts >= 8 && tiles * parts < 2 * slots + tiles)); parts++) {
            s.steps_per_part = steps > 0 ? (int)((steps + parts - 1) / parts) : 1;
            s.parts = steps > 0 ? (int)((steps + s.steps_per_part - 1) / s.steps_per_part) : 1;
            const double rounds = (double)((tiles * s.parts + slots - 1) / slots);
            double us = rounds * (s.steps_per_part * c.slice_us + 4.0);
            if (s.parts > 1) us += 4.0 + (2.0 * s.parts + 1) * (paired ? 2 : 1) * rows * cols * sizeof(T) / 4.5e6;
            if (best.parts == 0 || us < best_us) { best = s; best_us = us; }
        }
    }
    return best;
}
static uint64_t partial_elements(const Split& s, bool paired, int64_t rows, int64_t cols) {
    return s.parts > 1 ? (uint64_t)s.parts * (paired ? 2 : 1) * rows * cols : 0;
}

template <bool A_ALONG, bool B_ALONG, bool PAIRED, int EPI>
static void launch_tiles(Device* dev, const Product<float>& g, const Split& s, dim3 grid) {
    const auto run = [&](auto kernel, int threads) {
        const unsigned lds = 2 * 3 * (s.edge_m + s.edge_n) * 32;          // two buffers of three planes of both operands
        (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, dev->stream, g);
    };
    const auto go = [&](auto scaled) {
        constexpr bool S = decltype(scaled)::value;
        if (s.edge_n == 256)      run(split_product_kernel<S, 2, 4, 4, 2, A_ALONG, B_ALONG, PAIRED, EPI>, 512);
        else if (s.edge_m == 256) run(split_product_kernel<S, 4, 2, 2, 2, A_ALONG, B_ALONG, PAIRED, EPI>, 512);
        else                      run(split_product_kernel<S, 2, 2, 2, 2, A_ALONG, B_ALONG, PAIRED, EPI>, 256);
    };
    if (g.a_scale) go(std::true_type()); else go(std::false_type());
}
template <bool A_ALONG, bool B_ALONG, bool PAIRED, int EPI>
static void launch_tiles(Device* dev, const Product<double>& g, const Split&, dim3 grid) {
    // a matrix of one row lies along and across alike; taken as along, since the kernel reads what lies across by twos
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, dev->stream, g); };
    const bool a = A_ALONG || g.rows == 1, b = B_ALONG || g.cols == 1;
    if (a && b)  run(product_kernel<true, true, PAIRED, EPI>);
    else if (a)  run(product_kernel<true, false, PAIRED, EPI>);
    else if (b)  run(product_kernel<false, true, PAIRED, EPI>);
    else         run(product_kernel<false, false, PAIRED, EPI>);
}

template <typename T, bool PAIRED, int EPI>
static void launch_product(Device* dev, Product<T> g, const Split& s, bool a_along, bool b_along, T* partial) {
    g.tiles_m = s.tiles_m; g.tiles_n = s.tiles_n; g.steps_per_part = s.steps_per_part;
    const int64_t n = (int64_t)g.rows * g.cols;
    T* const out[3] = {g.out[0], g.out[1], g.out[2]};
    const dim3 grid((unsigned)(s.tiles_m * s.tiles_n * s.parts));
    const auto go = [&](auto epi) {
        constexpr int E = decltype(epi)::value;
        // (a transposed input only in the pair of weight gradients, where the errors lie by rows)
        if constexpr (PAIRED && E == STORE) { if (!a_along) { launch_tiles<false, false, PAIRED, E>(dev, g, s, grid); return; } }
        if (b_along) launch_tiles<true, true, PAIRED, E>(dev, g, s, grid);
        else         launch_tiles<true, false, PAIRED, E>(dev, g, s, grid);
    };
    if (s.parts == 1) { go(std::integral_constant<int, EPI>()); return; }
    g.out[0] = partial; g.out[1] = partial + n; g.out[2] = nullptr;
    g.part_stride = n * (PAIRED ? 2 : 1);
    go(std::integral_constant<int, STORE>());
    hipLaunchKernelGGL((product_join_kernel<T, PAIRED, EPI>), dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, dev->stream, partial, s.parts, n, g.fun, out[0], out[1], out[2]);
}

// The products of up to 64 rows: GATED, where both have the same A, or SUM, where each has its own.
struct FewPlan { int row_tiles, width, groups, parts, steps_per_part; };
template <typename T>
static FewPlan few_plan(const Device* dev, int64_t rows, int64_t cols, int64_t inner, bool along) {
    FewPlan f;
    const int64_t cus = dev->props.multiProcessorCount, chunk = 64 / (int64_t)sizeof(T), chunks = inner / chunk;
    f.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    f.width = sizeof(T) == 4 && f.row_tiles == 1 && !along && cols > 1 ? 2 : 1;
    f.groups = (int)((cols + 16 * f.width - 1) / (16 * f.width));
    // So many parts that the unit with the most blocks has the least to do (a hundredth of the whole charged for joining each), of at least
    // 16 chunks, which keep all wavefronts busy.
    int64_t parts = 1;
    const auto busiest = [&](int64_t p) { return (double)((f.groups * p + cus - 1) / cus) / p + 0.01 * p; };
    for (int64_t p = 2; p <= 16 && p <= chunks / 16 && f.groups < cus; p++)
        if (busiest(p) < busiest(parts)) parts = p;
    f.steps_per_part = chunks ? (int)((chunks + parts - 1) / parts) : 1;
    f.steps_per_part += f.steps_per_part & 1;                            // (chunks are taken in twos)
    f.parts = chunks ? (int)((chunks + f.steps_per_part - 1) / f.steps_per_part) : 1;
    return f;
}
// the parts' sums, in elements: whole fragments of 16 x 16
static uint64_t few_partial_elements(const FewPlan& f) { return f.parts > 1 ? (uint64_t)f.parts * f.groups * 2 * f.row_tiles * f.width * 256 : 0; }

template <typename T, int EPI>
static int launch_few(Device* dev, Product<T> g, const FewPlan& f, bool along, T* partial) {
    g.tiles_n = f.groups; g.steps_per_part = f.steps_per_part;
    unsigned* arrived = nullptr;
    if (f.parts > 1) {
        NK_REQUIRE((unsigned)f.groups <= ARRIVALS, "nk_gated_matmul: %d groups of columns share their sums, %u can", f.groups, ARRIVALS);
        if (int e = arrivals(dev, &arrived)) return e;
    }
    hipError_t refused = hipSuccess;
    const auto go = [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        const unsigned bytes = 8 * 2 * RT * f.width * 64 * 4 * sizeof(T);
        const auto run = [&](auto kernel) {
            if (bytes > 65536) refused = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
            if (refused == hipSuccess) hipLaunchKernelGGL(kernel, dim3((unsigned)(f.groups * f.parts)), dim3(512), bytes, dev->stream, g, f.parts, partial, arrived);
        };
        if (along) run(few_rows_kernel<T, RT, 1, true, EPI>);
        else if (f.width == 1) run(few_rows_kernel<T, RT, 1, false, EPI>);
        else if constexpr (sizeof(T) == 4 && RT == 1) run(few_rows_kernel<T, RT, 2, false, EPI>);
    };
    if (f.row_tiles == 1)      go(std::integral_constant<int, 1>());
    else if (f.row_tiles == 2) go(std::integral_constant<int, 2>());
    else                       go(std::integral_constant<int, 4>());
    NK_HIP(refused);
    return NK_OK;
}

// Whether a product takes two planes.  They save three of six partial products (at 1.1e15 operations a second) and cost a launch that reads
// both operands and a look at every result.  Forward in microseconds, weights that no cache holds, two planes against three:
// 512 x 1024 x 1024 33.7 / 29.2, 1024^3 40.4 / 38.8, 1111 x 1000 x 2500 73 / 97, 2048^3 153 / 208; 65 x 4096 x 4096, all weights, 92 / 63.
template <typename T> static bool two_planes(int64_t rows, int64_t cols, int64_t inner) {
    const double saved_us = 6.0 * rows * cols * inner / 1.1e9, cost_us = 9.0 + 4.0 * (rows + cols) * inner / 4.5e6;
    return sizeof(T) == 4 && saved_us > cost_us;
}
// Whether M rows go to few_rows_kernel.  Above 32 rows it holds four row tiles per wavefront and is bound by its matrix instructions, of
// which the tiles have faster ones (f32) or feed them better (f64): there only while the weights are few, where the tiles' slices are too
// short to fill the chip.  64 rows, weights by row, few rows / tiles in microseconds, forward and d_X: f32 1024 x 1024 (8 MB) 12 / 19 and
// 16 / 23, 2000 x 1500 (24 MB) 33 / 23 and 32 / 29; f64 700 x 150 (2 MB) 12 / 13 and 11 / 17, 300 x 2000 (10 MB) 14 / 16 and 34 / 23.
template <typename T> static bool takes_few_rows(int64_t M, int64_t K, int64_t N) {
    return M <= 32 || (M <= 64 && 2 * K * N * (int64_t)sizeof(T) < (sizeof(T) == 8 ? 5000000 : 20000000));
}
static void add_job(ScaleJobs& jobs, const float* p, const float* second, int64_t ld, int64_t count, int64_t length, bool along, int* out) {
    jobs.job[jobs.n++] = {{p, second}, ld, (int)count, (int)length, along, out, (unsigned)(along ? (count + 7) / 8 : (count + 31) / 32)};
}
static void launch_scales(Device* dev, const ScaleJobs& jobs) {
    unsigned blocks = 0;
    for (int i = 0; i < jobs.n; i++) blocks += jobs.job[i].blocks;
    hipLaunchKernelGGL(operand_scales_kernel, dim3(blocks), dim3(512), 0, dev->stream, jobs);
}

// What ran, for nk_last_path: f64 tiles, or those of two or three planes; split: the contraction in parts.
static int tiles_name(size_t item, bool two) { return item == 8 ? 0 : two ? 1 : 2; }
static const char* const TILES[3] = {"gated_tiles", "gated_tiles_two_planes", "gated_tiles_three_planes"};
static const char* const TILES_SPLIT[3] = {"gated_tiles_split", "gated_tiles_two_planes_split", "gated_tiles_three_planes_split"};
#define NK_BACKWARD_WITH(x) {"gated_backward" x, "gated_backward" x "_w_tiles", "gated_backward" x "_w_tiles_split", "gated_backward" x "_w_two_planes", \
                             "gated_backward" x "_w_two_planes_split", "gated_backward" x "_w_three_planes", "gated_backward" x "_w_three_planes_split"}
static const char* const BACKWARD[9][7] = {          // [d_X: not wanted, few rows, few rows split, then as the second][weights: not wanted, tiles, ...]
    NK_BACKWARD_WITH(""), NK_BACKWARD_WITH("_x_few_rows"), NK_BACKWARD_WITH("_x_few_rows_split"), NK_BACKWARD_WITH("_x_tiles"), NK_BACKWARD_WITH("_x_tiles_split"),
    NK_BACKWARD_WITH("_x_two_planes"), NK_BACKWARD_WITH("_x_two_planes_split"), NK_BACKWARD_WITH("_x_three_planes"), NK_BACKWARD_WITH("_x_three_planes_split")};
#undef NK_BACKWARD_WITH

template <typename T>
static int gated_forward(Device* dev, int fun, bool along, int64_t M, int64_t K, int64_t N, const T* X, const T* Wg, const T* Wu, T* H, T* gate, T* up) {
    Product<T> g{};
    g.A[0] = X; g.lda = K; g.B[0] = Wg; g.B[1] = Wu; g.ldb = along ? K : N;
    g.rows = (int)M; g.cols = (int)N; g.inner = (int)K; g.segments = 1; g.fun = fun;
    g.out[0] = H; g.out[1] = gate; g.out[2] = up;
    void* ws = nullptr;
    if (takes_few_rows<T>(M, K, N)) {
        const FewPlan f = few_plan<T>(dev, M, N, K, along);
        if (const uint64_t need = few_partial_elements(f))
            if (int e = workspace(dev, need * sizeof(T), &ws)) return e;
        if (int e = launch_few<T, GATED>(dev, g, f, along, (T*)ws)) return e;
        NK_HIP(hipGetLastError());
        set_path(f.parts > 1 ? "gated_few_rows_split" : "gated_few_rows");
        return NK_OK;
    }
    const Split s = plan<T>(dev, true, M, N, K, 1);
    const bool two = two_planes<T>(M, 2 * N, K);
    const uint64_t parts_bytes = partial_elements(s, true, M, N) * sizeof(T), need = parts_bytes + (two ? (M + 2 * N) * sizeof(int) : 0);
    if (need) if (int e = workspace(dev, need, &ws)) return e;
    if constexpr (sizeof(T) == 4) if (two) {
        int* const scales = (int*)((char*)ws + parts_bytes);
        ScaleJobs jobs{};
        add_job(jobs, X, nullptr, K, M, K, true, scales);
        add_job(jobs, Wg, nullptr, g.ldb, N, K, along, scales + M);
        add_job(jobs, Wu, nullptr, g.ldb, N, K, along, scales + M + N);
        launch_scales(dev, jobs);
        g.a_scale = scales; g.b_scale[0] = scales + M; g.b_scale[1] = scales + M + N;
    }
    launch_product<T, true, GATED>(dev, g, s, true, along, (T*)ws);
    NK_HIP(hipGetLastError());
    const int t = tiles_name(sizeof(T), two);
    set_path(s.parts > 1 ? TILES_SPLIT[t] : TILES[t]);
    return NK_OK;
}

template <typename T>
static int gated_backward(Device* dev, int fun, bool along, int64_t M, int64_t K, int64_t N, const T* X, const T* Wg, const T* Wu, const T* gate, const T* up,
                          const T* E, T* dX, T* dWg, T* dWu) {
    const int64_t n = M * N;
    const Split sx = plan<T>(dev, false, M, K, N, 2), sw = plan<T>(dev, true, K, N, M, 1);
    const FewPlan few = few_plan<T>(dev, M, K, N, !along);
    const bool is_few = takes_few_rows<T>(M, K, N);
    const uint64_t px = dX ? is_few ? few_partial_elements(few) : partial_elements(sx, false, M, K) : 0, pw = dWg ? partial_elements(sw, true, K, N) : 0;
    const bool two_x = dX && !is_few && two_planes<T>(M, K, 2 * N), two_w = dWg && two_planes<T>(K, 2 * N, M);
    const uint64_t scales_x = two_x ? M + K : 0, scales_w = two_w ? K + 2 * N : 0;
    void* ws = nullptr;
    const uint64_t room = (2 * (uint64_t)n + 15) & ~(uint64_t)15;            // both errors; what follows starts at a whole vector
    if (int e = workspace(dev, (room + (px > pw ? px : pw)) * sizeof(T) + (scales_x + scales_w) * sizeof(int), &ws)) return e;
    T *const dg = (T*)ws, *const du = dg + n, *const partial = dg + room;
    hipLaunchKernelGGL((gated_errors_kernel<T>), dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, dev->stream, fun, n, E, gate, up, dg, du);
    Product<T> gx{}, gw{};
    gx.A[0] = dg; gx.A[1] = du; gx.lda = N; gx.B[0] = Wg; gx.B[1] = Wu; gx.ldb = along ? K : N;      // (weights stored by row have neighbours along N)
    gx.rows = (int)M; gx.cols = (int)K; gx.inner = (int)N; gx.segments = 2;
    gx.out[0] = dX;
    gw.A[0] = X; gw.lda = K; gw.B[0] = dg; gw.B[1] = du; gw.ldb = N;
    gw.rows = (int)K; gw.cols = (int)N; gw.inner = (int)M; gw.segments = 1;
    gw.out[0] = dWg; gw.out[1] = dWu;
    if constexpr (sizeof(T) == 4) {
        int *const scales = (int*)(partial + (px > pw ? px : pw)), *const at = scales + scales_x;
        ScaleJobs jobs{};
        if (two_x) {
            add_job(jobs, dg, du, N, M, N, true, scales);
            add_job(jobs, Wg, Wu, gx.ldb, K, N, !along, scales + M);
            gx.a_scale = scales; gx.b_scale[0] = scales + M;
        }
        if (two_w) {
            add_job(jobs, X, nullptr, K, K, M, false, at);
            add_job(jobs, dg, nullptr, N, N, M, false, at + K);
            add_job(jobs, du, nullptr, N, N, M, false, at + K + N);
            gw.a_scale = at; gw.b_scale[0] = at + K; gw.b_scale[1] = at + K + N;
        }
        if (jobs.n) launch_scales(dev, jobs);
    }
    if (dX) {
        if (is_few) { if (int e = launch_few<T, SUM>(dev, gx, few, !along, partial)) return e; }
        else launch_product<T, false, STORE>(dev, gx, sx, true, !along, partial);
    }
    if (dWg) launch_product<T, true, STORE>(dev, gw, sw, false, false, partial);
    NK_HIP(hipGetLastError());
    const int x = !dX ? 0 : is_few ? 1 + (few.parts > 1) : 3 + 2 * tiles_name(sizeof(T), two_x) + (sx.parts > 1);
    const int w = !dWg ? 0 : 1 + 2 * tiles_name(sizeof(T), two_w) + (sw.parts > 1);
    set_path(BACKWARD[x][w]);
    return NK_OK;
}

static int check_gated(const char* what, int fun, int dtype, int layout, int64_t M, int64_t K, int64_t N) {
    NK_REQUIRE(dtype == NK_F32 || dtype == NK_F64, "%s: unknown dtype %d", what, dtype);
    NK_REQUIRE(fun == NK_FUN_IDY || fun == NK_FUN_RELU || fun == NK_FUN_SIG || fun == NK_FUN_SILU || fun == NK_FUN_GELU || fun == NK_FUN_TANH,
               "%s: function id %d is none of idy, relu, sig, silu, gelu, tanh", what, fun);
    NK_REQUIRE(layout == NK_LAYOUT_ROW_MAJOR || layout == NK_LAYOUT_COLUMN_MAJOR, "%s: unknown layout %d", what, layout);
    const int64_t most = (int64_t)1 << 31, longest = ((int64_t)1 << 27) - 1024;       // (512 threads for 16 of an axis stay below the 2^32 of a launch)
    NK_REQUIRE(M >= 1 && K >= 1 && N >= 1, "%s: M, K, N must be positive (got %lld, %lld, %lld)", what, (long long)M, (long long)K, (long long)N);
    NK_REQUIRE(M <= longest && K <= longest && N <= longest && M * K < most && K * N < most && M * N < most, "%s: operands are limited to 2^31-1 elements and axes to 2^27-1024", what);
    return NK_OK;
}
struct Piece { const char* name; nk_buf at; uint64_t bytes; };
// every piece inside a live buffer, and no output (the last `outputs` pieces) on another piece
static int check_pieces(Device* dev, const char* what, const Piece* p, int count, int outputs, uint64_t element) {
    for (int i = 0; i < count; i++) {
        if (!p[i].at && i >= count - outputs) continue;
        NK_REQUIRE(p[i].at % element == 0, "%s: %s does not start at an element", what, p[i].name);
        if (int e = check_range(dev, p[i].name, p[i].at, 0, p[i].bytes)) return e;
    }
    for (int i = count - outputs; i < count; i++)
        for (int j = 0; j < i; j++)
            NK_REQUIRE(!p[i].at || !p[j].at || p[i].at >= p[j].at + p[j].bytes || p[j].at >= p[i].at + p[i].bytes, "%s: %s overlaps %s", what, p[i].name, p[j].name);
    return NK_OK;
}

}  // namespace nk

using namespace nk;

extern "C" int nk_gated_matmul(nk_dev h, int fun, int dtype, int layout, int64_t M, int64_t K, int64_t N, nk_buf X, nk_buf Wg, nk_buf Wu,
                               nk_buf drn, nk_buf gate, nk_buf up) {
    NK_DEVICE(dev, h);
    const char* what = "nk_gated_matmul";
    if (int e = check_gated(what, fun, dtype, layout, M, K, N)) return e;
    NK_REQUIRE(drn != 0, "%s: no drain", what);
    NK_REQUIRE((gate == 0) == (up == 0), "%s: gate and up are kept together or not at all", what);
    const uint64_t eb = dtype_bytes(dtype), x = M * K * eb, w = K * N * eb, y = M * N * eb;
    const Piece p[] = {{"X", X, x}, {"Wg", Wg, w}, {"Wu", Wu, w}, {"the drain", drn, y}, {"gate", gate, y}, {"up", up, y}};
    if (int e = check_pieces(dev, what, p, 6, 3, eb)) return e;
    const bool along = layout == NK_LAYOUT_COLUMN_MAJOR;
    return dtype == NK_F32 ? gated_forward<float>(dev, fun, along, M, K, N, (const float*)X, (const float*)Wg, (const float*)Wu, (float*)drn, (float*)gate, (float*)up)
                           : gated_forward<double>(dev, fun, along, M, K, N, (const double*)X, (const double*)Wg, (const double*)Wu, (double*)drn, (double*)gate, (double*)up);
}

extern "C" int nk_gated_matmul_backward(nk_dev h, int fun, int dtype, int layout, int64_t M, int64_t K, int64_t N, nk_buf X, nk_buf Wg, nk_buf Wu,
                                        nk_buf gate, nk_buf up, nk_buf error, nk_buf dX, nk_buf dWg, nk_buf dWu) {
    NK_DEVICE(dev, h);
    const char* what = "nk_gated_matmul_backward";
    if (int e = check_gated(what, fun, dtype, layout, M, K, N)) return e;
    NK_REQUIRE(dX || dWg, "%s: no gradient is asked for", what);
    NK_REQUIRE((dWg == 0) == (dWu == 0), "%s: the gradients of the weights are computed together or not at all", what);
    const uint64_t eb = dtype_bytes(dtype), x = M * K * eb, w = K * N * eb, y = M * N * eb;
    const Piece p[] = {{"X", X, x}, {"Wg", Wg, w}, {"Wu", Wu, w}, {"gate", gate, y}, {"up", up, y}, {"error", error, y}, {"d_X", dX, x}, {"d_Wg", dWg, w}, {"d_Wu", dWu, w}};
    if (int e = check_pieces(dev, what, p, 9, 3, eb)) return e;
    const bool along = layout == NK_LAYOUT_COLUMN_MAJOR;
    return dtype == NK_F32 ? gated_backward<float>(dev, fun, along, M, K, N, (const float*)X, (const float*)Wg, (const float*)Wu, (const float*)gate, (const float*)up,
                                                   (const float*)error, (float*)dX, (float*)dWg, (float*)dWu)
                           : gated_backward<double>(dev, fun, along, M, K, N, (const double*)X, (const double*)Wg, (const double*)Wu, (const double*)gate, (const double*)up,
                                                    (const double*)error, (double*)dX, (double*)dWg, (double*)dWu);
}
