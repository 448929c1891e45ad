// nk_gated_matmul, nk_gated_matmul_backward: the gated half of a feed-forward block.
//
//     gate = X Wg      up = X Wu      H = f(gate) up
//     with the error E of H:  dg = E up f'(gate)   du = E f(gate)   dX = dg Wg^T + du Wu^T   dWg = X^T dg   dWu = X^T du
//
// All products are one kernel, result(m, n) = sum over l of A(m, l) B(n, l), on tiles of the result whose operands pass through
// LDS.  Two switches say where an operand's neighbours along l lie (next to each other, or a row apart), which covers X, its
// transpose and weights of either layout without a copy.  Two products that share A (forward, weight gradients) are
// PAIRED: a tile holds the same columns of both, half each, so that A is staged once for both and f(gate) up is formed in the
// registers that hold the sums.  dX is one product over a contraction of two segments, (dg, Wg) and then (du, Wu).
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
    T* out[3];                          // GATED: H, gate, up; STORE: the product (both halves)
};
enum { STORE = 0, GATED = 1 };

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
__device__ __forceinline__ void own_tile(unsigned block, unsigned tiles, int tiles_m, int tiles_n, int& tm, int& tn) {
    const unsigned each = tiles / 8, rest = tiles % 8, xcd = block % 8, at = block / 8;
    const unsigned id = xcd * each + (xcd < rest ? xcd : rest) + at;
    const unsigned band = 8 * (unsigned)tiles_n, b = id / band, in = id - b * band;
    const unsigned height = (unsigned)tiles_m - b * 8 < 8 ? (unsigned)tiles_m - b * 8 : 8;
    tm = (int)(b * 8 + in % height);
    tn = (int)(in / height);
}

// One operand's share of a slice: `WIDTH` rows of the result (or columns, for B) by 16 steps of l, 256 threads, E consecutive l each.
template <typename T, int WIDTH, bool ALONG>
struct Share {
    static constexpr int BK = 16, E = WIDTH * BK / 256, PER_ROW = BK / E;
    T v[E];
    // `row`: the operand's first element of this thread's row; `l0`: the slice's first l
    static __device__ __forceinline__ int row_of(int t) { return ALONG ? t / PER_ROW : t % WIDTH; }
    static __device__ __forceinline__ int l_of(int t) { return (ALONG ? t % PER_ROW : t / WIDTH) * E; }
    __device__ __forceinline__ void load(const T* row, int64_t ld, int l0, int inner, int t) {
        const int l = l0 + l_of(t);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = l + e < inner ? row[(int64_t)(l + e) * (ALONG ? 1 : ld)] : T(0);
    }
    // LDS: fragments of 16 rows x 4 l, in the order in which the lanes of a wavefront hold them
    __device__ __forceinline__ void store(T* lds, int t) const {
        const int r = row_of(t), l = l_of(t);
#pragma unroll
        for (int e = 0; e < E; e++) lds[((r >> 4) * (BK / 4) + ((l + e) >> 2)) * 64 + ((l + e) & 3) * 16 + (r & 15)] = v[e];
    }
};

// 128 x 128 tiles, 4 wavefronts of 64 x 64, slices of 16 l in two LDS buffers.  f64: 64 x 64 x 16 multiply-adds are 16 x 4 matrix
// instructions against 32 LDS reads of 8 bytes a lane.
template <typename T, bool A_ALONG, bool B_ALONG, bool PAIRED, int EPI>
__global__ __launch_bounds__(256) void product_kernel(const Product<T> g) {
    typedef Quad<T> Q;
    typedef typename Q::Acc Acc;
    constexpr int BM = 128, BN = 128, BK = 16;
    __shared__ T a_lds[2][BM * BK], b_lds[2][BN * BK];
    const unsigned tiles = (unsigned)(g.tiles_m * g.tiles_n), part = blockIdx.x / tiles;
    int tm, tn;
    own_tile(blockIdx.x - part * tiles, tiles, g.tiles_m, g.tiles_n, tm, tn);
    constexpr int HALF = PAIRED ? BN / 2 : BN;
    const int m0 = tm * BM, n0 = tn * HALF;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, wm = wave >> 1, wn = wave & 1;
    Share<T, BM, A_ALONG> a;
    Share<T, BN, B_ALONG> b;
    // rows and columns past the end are read as the last one; what they give is not stored
    const int64_t am = m0 + a.row_of(t) < g.rows ? m0 + a.row_of(t) : g.rows - 1;
    const int bt = b.row_of(t), half = PAIRED ? bt / HALF : 0, bc = n0 + (PAIRED ? bt % HALF : bt);
    const int64_t bn = bc < g.cols ? bc : g.cols - 1;
    const int per_segment = (g.inner + BK - 1) / BK;
    const int first = (int)part * g.steps_per_part, all = per_segment * g.segments;
    const int last = first + g.steps_per_part < all ? first + g.steps_per_part : all;
    const auto request = [&](int s) {
        const int segment = s / per_segment, l0 = (s - segment * per_segment) * BK;
        a.load(g.A[segment] + am * (A_ALONG ? g.lda : 1), g.lda, l0, g.inner, t);
        b.load(g.B[PAIRED ? half : segment] + bn * (B_ALONG ? g.ldb : 1), g.ldb, l0, g.inner, t);
    };
    Acc acc[4][4] = {};
    request(first);
    a.store(a_lds[0], t); b.store(b_lds[0], t);
    if (first + 1 < last) request(first + 1);
    __syncthreads();
    for (int s = first; s < last; s++) {
        const int cur = (s - first) & 1;
        const T *const ap = a_lds[cur] + lane, *const bp = b_lds[cur] + lane;
#pragma unroll
        for (int k = 0; k < BK / 4; k++) {
            T af[4], bf[4];
#pragma unroll
            for (int i = 0; i < 4; i++) af[i] = ap[((wm * 4 + i) * (BK / 4) + k) * 64];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int block = PAIRED ? (j >> 1) * 4 + wn * 2 + (j & 1) : wn * 4 + j;
                bf[j] = bp[(block * (BK / 4) + k) * 64];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = Q::mma(af[i], bf[j], acc[i][j]);
        }
        if (s + 1 < last) {
            a.store(a_lds[cur ^ 1], t); b.store(b_lds[cur ^ 1], t);
            if (s + 2 < last) request(s + 2);
        }
        __syncthreads();
    }
    const int64_t shift = (int64_t)part * g.part_stride;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int m = m0 + wm * 64 + i * 16 + Q::row(lane, v);
            if (m >= g.rows) continue;
            const int64_t row = (int64_t)m * g.cols + shift;
#pragma unroll
            for (int j = 0; j < (PAIRED ? 2 : 4); j++) {
                const int n = n0 + (PAIRED ? wn * 32 : wn * 64) + j * 16 + (lane & 15);
                if (n >= g.cols) continue;
                const T x = acc[i][j][v];
                if constexpr (!PAIRED) g.out[0][row + n] = x;
                else {
                    const T y = acc[i][2 + (j & 1)][v];
                    if constexpr (EPI == GATED) {
                        g.out[0][row + n] = gated_fun(g.fun, x) * y;
                        if (g.out[1]) { g.out[1][row + n] = x; g.out[2][row + n] = y; }
                    } else { g.out[0][row + n] = x; g.out[1][row + n] = y; }
                }
            }
        }
}

// ---- parts of the contraction, added in order -----------------------------------------------------------------------
// partial: [parts][halves][n]; halves 2: the pair of products
template <typename T, bool PAIRED, int EPI>
__global__ __launch_bounds__(256) void product_join_kernel(const T* __restrict__ partial, int parts, int64_t n, int fun, T* out0, T* out1, T* out2) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    constexpr int HALVES = PAIRED ? 2 : 1;
    T x = partial[i], y = PAIRED ? partial[n + i] : T(0);
    for (int p = 1; p < parts; p++) {
        x += partial[(int64_t)p * HALVES * n + i];
        if (PAIRED) y += partial[((int64_t)p * HALVES + 1) * n + i];
    }
    if constexpr (EPI == GATED) {
        out0[i] = gated_fun(fun, x) * y;
        if (out1) { out1[i] = x; out2[i] = y; }
    } else {
        out0[i] = x;
        if (PAIRED) out1[i] = y;
    }
}

// dg = E up f'(gate), du = E f(gate)
template <typename T>
__global__ __launch_bounds__(256) void gated_errors_kernel(int fun, int64_t n, const T* __restrict__ error, const T* __restrict__ gate, const T* __restrict__ up,
                                                           T* __restrict__ d_gate, T* __restrict__ d_up) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    T f, slope;
    gated_fun_and_slope(fun, gate[i], f, slope);
    d_gate[i] = error[i] * up[i] * slope;
    d_up[i] = error[i] * f;
}

// ---- plans ---------------------------------------------------------------------------------------------------------------
struct Split { int tiles_m, tiles_n, parts, steps_per_part; };
static Split plan(const Device* dev, bool paired, int64_t rows, int64_t cols, int64_t inner, int segments) {
    Split s;
    s.tiles_m = (int)((rows + 127) / 128);
    s.tiles_n = (int)(paired ? (cols + 63) / 64 : (cols + 127) / 128);
    const int64_t tiles = (int64_t)s.tiles_m * s.tiles_n, steps = (inner + 15) / 16 * segments, want = 2 * dev->props.multiProcessorCount;
    int64_t parts = tiles >= want ? 1 : want / tiles;
    if (parts > steps / 8) parts = steps / 8 > 0 ? steps / 8 : 1;
    s.steps_per_part = (int)((steps + parts - 1) / parts);
    s.parts = (int)((steps + s.steps_per_part - 1) / s.steps_per_part);
    return s;
}
static uint64_t partial_elements(const Split& s, bool paired, int64_t rows, int64_t cols) {
    return s.parts > 1 ? (uint64_t)s.parts * (paired ? 2 : 1) * rows * cols : 0;
}

template <typename T, bool PAIRED, int EPI>
static void launch_product(Device* dev, Product<T> g, const Split& s, bool a_along, bool b_along, T* partial) {
    g.tiles_m = s.tiles_m; g.tiles_n = s.tiles_n; g.steps_per_part = s.steps_per_part;
    const int64_t n = (int64_t)g.rows * g.cols;
    T* const out[3] = {g.out[0], g.out[1], g.out[2]};
    const dim3 grid((unsigned)(s.tiles_m * s.tiles_n * s.parts));
    const auto go = [&](auto epi) {
        constexpr int E = decltype(epi)::value;
        if (a_along && b_along)       hipLaunchKernelGGL((product_kernel<T, true, true, PAIRED, E>), grid, dim3(256), 0, dev->stream, g);
        else if (a_along)             hipLaunchKernelGGL((product_kernel<T, true, false, PAIRED, E>), grid, dim3(256), 0, dev->stream, g);
        else                          hipLaunchKernelGGL((product_kernel<T, false, false, PAIRED, E>), grid, dim3(256), 0, dev->stream, g);
    };
    if (s.parts == 1) { go(std::integral_constant<int, EPI>()); return; }
    g.out[0] = partial; g.out[1] = partial + n; g.out[2] = nullptr;
    g.part_stride = n * (PAIRED ? 2 : 1);
    go(std::integral_constant<int, STORE>());
    hipLaunchKernelGGL((product_join_kernel<T, PAIRED, EPI>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, dev->stream, partial, s.parts, n, g.fun, out[0], out[1], out[2]);
}

template <typename T>
static int gated_forward(Device* dev, int fun, bool along, int64_t M, int64_t K, int64_t N, const T* X, const T* Wg, const T* Wu, T* H, T* gate, T* up) {
    Product<T> g{};
    g.A[0] = X; g.lda = K; g.B[0] = Wg; g.B[1] = Wu; g.ldb = along ? K : N;
    g.rows = (int)M; g.cols = (int)N; g.inner = (int)K; g.segments = 1; g.fun = fun;
    g.out[0] = H; g.out[1] = gate; g.out[2] = up;
    const Split s = plan(dev, true, M, N, K, 1);
    void* ws = nullptr;
    if (const uint64_t need = partial_elements(s, true, M, N))
        if (int e = workspace(dev, need * sizeof(T), &ws)) return e;
    launch_product<T, true, GATED>(dev, g, s, true, along, (T*)ws);
    NK_HIP(hipGetLastError());
    set_path(s.parts > 1 ? "gated_tiles_split" : "gated_tiles");
    return NK_OK;
}

template <typename T>
static int gated_backward(Device* dev, int fun, bool along, int64_t M, int64_t K, int64_t N, const T* X, const T* Wg, const T* Wu, const T* gate, const T* up,
                          const T* E, T* dX, T* dWg, T* dWu) {
    const int64_t n = M * N;
    const Split sx = plan(dev, false, M, K, N, 2), sw = plan(dev, true, K, N, M, 1);
    const uint64_t px = dX ? partial_elements(sx, false, M, K) : 0, pw = dWg ? partial_elements(sw, true, K, N) : 0;
    void* ws = nullptr;
    if (int e = workspace(dev, (2 * (uint64_t)n + (px > pw ? px : pw)) * sizeof(T), &ws)) return e;
    T *const dg = (T*)ws, *const du = dg + n, *const partial = du + n;
    hipLaunchKernelGGL((gated_errors_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, dev->stream, fun, n, E, gate, up, dg, du);
    if (dX) {
        Product<T> g{};
        g.A[0] = dg; g.A[1] = du; g.lda = N; g.B[0] = Wg; g.B[1] = Wu; g.ldb = along ? K : N;
        g.rows = (int)M; g.cols = (int)K; g.inner = (int)N; g.segments = 2;
        g.out[0] = dX;
        launch_product<T, false, STORE>(dev, g, sx, true, !along, partial);      // (weights stored by row have neighbours along N)
    }
    if (dWg) {
        Product<T> g{};
        g.A[0] = X; g.lda = K; g.B[0] = dg; g.B[1] = du; g.ldb = N;
        g.rows = (int)K; g.cols = (int)N; g.inner = (int)M; g.segments = 1;
        g.out[0] = dWg; g.out[1] = dWu;
        launch_product<T, true, STORE>(dev, g, sw, false, false, partial);
    }
    NK_HIP(hipGetLastError());
    set_path("gated_backward_tiles");
    return NK_OK;
}

static int check_gated(const char* what, int fun, int dtype, int layout, int64_t M, int64_t K, int64_t N) {
    NK_REQUIRE(dtype == NK_F32 || dtype == NK_F64, "%s: unknown dtype %d", what, dtype);
    NK_REQUIRE(fun == NK_FUN_IDY || fun == NK_FUN_RELU || fun == NK_FUN_SIG || fun == NK_FUN_SILU || fun == NK_FUN_GELU || fun == NK_FUN_TANH,
               "%s: function id %d is none of idy, relu, sig, silu, gelu, tanh", what, fun);
    NK_REQUIRE(layout == NK_LAYOUT_ROW_MAJOR || layout == NK_LAYOUT_COLUMN_MAJOR, "%s: unknown layout %d", what, layout);
    const int64_t most = (int64_t)1 << 31;
    NK_REQUIRE(M >= 1 && K >= 1 && N >= 1, "%s: M, K, N must be positive (got %lld, %lld, %lld)", what, (long long)M, (long long)K, (long long)N);
    NK_REQUIRE(M < most && K < most && N < most && M * K < most && K * N < most && M * N < most, "%s: operands are limited to 2^31-1 elements", what);
    return NK_OK;
}
struct Piece { const char* name; nk_buf at; uint64_t bytes; };
// every piece inside a live buffer, and no output (the last `outputs` pieces) on another piece
static int check_pieces(Device* dev, const char* what, const Piece* p, int count, int outputs) {
    for (int i = 0; i < count; i++) {
        if (!p[i].at && i >= count - outputs) continue;
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
    if (int e = check_pieces(dev, what, p, 6, 3)) return e;
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
    if (int e = check_pieces(dev, what, p, 9, 3)) return e;
    const bool along = layout == NK_LAYOUT_COLUMN_MAJOR;
    return dtype == NK_F32 ? gated_backward<float>(dev, fun, along, M, K, N, (const float*)X, (const float*)Wg, (const float*)Wu, (const float*)gate, (const float*)up,
                                                   (const float*)error, (float*)dX, (float*)dWg, (float*)dWu)
                           : gated_backward<double>(dev, fun, along, M, K, N, (const double*)X, (const double*)Wg, (const double*)Wu, (const double*)gate, (const double*)up,
                                                    (const double*)error, (double*)dX, (double*)dWg, (double*)dWu);
}
