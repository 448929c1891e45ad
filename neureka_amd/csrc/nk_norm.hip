// nk_layer_norm, nk_layer_norm_backward: every row of a matrix brought to mean 0 and variance 1, times a gain, plus a bias.
//
//     mean = sum x / D      var = sum (x - mean)^2 / D      rstd = 1 / sqrt(var + epsilon)      h = (x - mean) rstd
//     y = h gain + bias
//     with the error e of y and g = e gain:
//     dx = rstd (g - sum g / D - h sum (g h) / D)      dgain = sum over rows of e h      dbias = sum over rows of e
//
// A row is read once: it stays in the registers of its group of threads (a wavefront up to 512 floats, a block of 256 or
// 1024 threads above) while its mean, then the sum of the squared distances from it, are formed; the variance is never
// a difference of two large sums.  A block keeps its columns' gain (and bias) in registers and walks over rows with the next row
// already requested.  The backward pass keeps the columns' share of dgain and dbias in registers as well and writes one
// partial row per block; a second launch adds the partial rows front to back, so the result does not depend on the order in
// which blocks run.  Rows that fit no block's registers are read once per pass.  All of it is bound by memory: two numbers per element
// forward, three backward.  Everything is computed in the element type.
#include "nk_internal.h"

namespace nk {

template <typename T> struct Wide {                          // 16 bytes; rows start at any element
    static constexpr int N = 16 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

__device__ __forceinline__ float root(float x) { return ::sqrtf(x); }
__device__ __forceinline__ double root(double x) { return ::sqrt(x); }
__device__ __forceinline__ float mul_add(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double mul_add(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Sums of `N` values over the THREADS threads that share a row, the same in every thread.
template <typename T, int THREADS, int N>
__device__ __forceinline__ void row_sums(T (&s)[N], T* scratch) {
#pragma unroll
    for (int step = 32; step > 0; step >>= 1)
#pragma unroll
        for (int k = 0; k < N; k++) s[k] += __shfl_xor(s[k], step);
    if constexpr (THREADS > 64) {
        constexpr int WAVES = THREADS / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; k++) scratch[k * WAVES + wave] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            T sum = scratch[k * WAVES];
#pragma unroll
            for (int w = 1; w < WAVES; w++) sum += scratch[k * WAVES + w];
            s[k] = sum;
        }
        // the callers alternate between two scratch areas, so the next sums cannot overwrite these before all have read them
    }
}

// The vectors of one row that belong to a thread: vector v covers columns (v * THREADS + t) * N ...
template <typename T, int THREADS, int NV>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int cols, int t, typename Wide<T>::V (&x)[NV]) {
    constexpr int N = Wide<T>::N;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = (v * THREADS + t) * N;
        if (c + N <= cols) x[v] = *(const typename Wide<T>::V*)(row + c);
        else
#pragma unroll
            for (int e = 0; e < N; e++) x[v][e] = c + e < cols ? row[c + e] : T(0);
    }
}
template <typename T, int THREADS, int NV>
__device__ __forceinline__ void store_row(T* row, int cols, int t, const typename Wide<T>::V (&x)[NV]) {
    constexpr int N = Wide<T>::N;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = (v * THREADS + t) * N;
        if (c + N <= cols) *(typename Wide<T>::V*)(row + c) = x[v];
        else
#pragma unroll
            for (int e = 0; e < N; e++) if (c + e < cols) row[c + e] = x[v][e];
    }
}

template <typename T>
struct NormArgs {
    const T* src; int64_t pitch;                            // elements from one row to the next
    int64_t rows; int cols;
    const T* gain; const T* bias;
    T epsilon;
    T* drn; T* mean; T* rstd;                               // mean / rstd: written forward where not null, read backward
    const T* error;
    T* d_src;                                               // backward: null where not wanted
    T* partial;                                             // [2][blocks][cols]: shares of dgain, then of dbias; null where neither is wanted
};

// A block of BLOCK threads holds BLOCK / THREADS rows at a time, each in the registers of THREADS threads.
template <typename T, int BLOCK, int THREADS, int NV>
__global__ __launch_bounds__(BLOCK) void norm_forward_kernel(const NormArgs<T> a) {
    typedef typename Wide<T>::V V;
    constexpr int N = Wide<T>::N, GROUPS = BLOCK / THREADS;
    __shared__ T scratch[2][16];
    const int t = threadIdx.x % THREADS;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / THREADS;
    // (GROUPS > 1: a row belongs to one wavefront, there is no barrier in the loop and wavefronts may leave it at different times)
    if (row >= a.rows) return;
    V x[NV], gain[NV], bias[NV];
    load_row<T, THREADS, NV>(a.src + row * a.pitch, a.cols, t, x);
    load_row<T, THREADS, NV>(a.gain, a.cols, t, gain);
    load_row<T, THREADS, NV>(a.bias, a.cols, t, bias);
    const T count = T(a.cols);
    for (; row < a.rows; row += step) {
        V next[NV];
        const bool more = row + step < a.rows;
        if (more) load_row<T, THREADS, NV>(a.src + (row + step) * a.pitch, a.cols, t, next);
        T s[1] = {T(0)};
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int e = 0; e < N; e++) s[0] += x[v][e];
        row_sums<T, THREADS, 1>(s, scratch[0]);
        const T mean = s[0] / count;
        s[0] = T(0);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = (v * THREADS + t) * N;
#pragma unroll
            for (int e = 0; e < N; e++) {
                x[v][e] = x[v][e] - mean;
                if (c + e < a.cols) s[0] = mul_add(x[v][e], x[v][e], s[0]);
            }
        }
        row_sums<T, THREADS, 1>(s, scratch[1]);
        const T rstd = T(1) / root(s[0] / count + a.epsilon);
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int e = 0; e < N; e++) x[v][e] = mul_add(x[v][e] * rstd, gain[v][e], bias[v][e]);
        store_row<T, THREADS, NV>(a.drn + row * a.cols, a.cols, t, x);
        if (t == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
        if (more)
#pragma unroll
            for (int v = 0; v < NV; v++) x[v] = next[v];
    }
}

template <typename T, int BLOCK, int THREADS, int NV>
__global__ __launch_bounds__(BLOCK) void norm_backward_kernel(const NormArgs<T> a) {
    typedef typename Wide<T>::V V;
    constexpr int N = Wide<T>::N, GROUPS = BLOCK / THREADS;
    __shared__ T scratch[2][2 * 16];
    __shared__ T share[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? 64 * NV * N : 1];
    const int t = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    V gain[NV], dgain[NV], dbias[NV], x[NV], err[NV];
    load_row<T, THREADS, NV>(a.gain, a.cols, t, gain);
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
        for (int e = 0; e < N; e++) dgain[v][e] = dbias[v][e] = T(0);
    T mean = T(0), rstd = T(0);
    if (row < a.rows) {
        load_row<T, THREADS, NV>(a.src + row * a.pitch, a.cols, t, x);
        load_row<T, THREADS, NV>(a.error + row * a.cols, a.cols, t, err);
        mean = a.mean[row]; rstd = a.rstd[row];
    }
    const T count = T(a.cols);
    // a block of 1024 threads has 128 registers per thread: with four vectors of a row each, the next row does not fit beside this one (doubles
    // spill 38 registers even so)
    constexpr bool AHEAD = BLOCK < 1024 || NV < 4;
    for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
        V x_next[AHEAD ? NV : 1], err_next[AHEAD ? NV : 1];
        T mean_next = T(0), rstd_next = T(0);
        const bool more = row + step < a.rows;
        if (more) {
            if constexpr (AHEAD) {
                load_row<T, THREADS, NV>(a.src + (row + step) * a.pitch, a.cols, t, x_next);
                load_row<T, THREADS, NV>(a.error + (row + step) * a.cols, a.cols, t, err_next);
            }
            mean_next = a.mean[row + step]; rstd_next = a.rstd[row + step];
        }
        T s[2] = {T(0), T(0)};                              // of g and of g h; columns past the end have gain 0 and error 0
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = (v * THREADS + t) * N;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const T h = c + e < a.cols ? (x[v][e] - mean) * rstd : T(0);
                x[v][e] = h;
                dgain[v][e] = mul_add(err[v][e], h, dgain[v][e]);
                dbias[v][e] += err[v][e];
                const T g = err[v][e] * gain[v][e];
                err[v][e] = g;
                s[0] += g;
                s[1] = mul_add(g, h, s[1]);
            }
        }
        if (a.d_src) {
            row_sums<T, THREADS, 2>(s, scratch[turn]);
            const T g_mean = s[0] / count, gh_mean = s[1] / count;
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int e = 0; e < N; e++) x[v][e] = rstd * (err[v][e] - mul_add(x[v][e], gh_mean, g_mean));
            store_row<T, THREADS, NV>(a.d_src + row * a.cols, a.cols, t, x);
        }
        if (more) {
            if constexpr (AHEAD) {
#pragma unroll
                for (int v = 0; v < NV; v++) { x[v] = x_next[v]; err[v] = err_next[v]; }
            } else {
                load_row<T, THREADS, NV>(a.src + (row + step) * a.pitch, a.cols, t, x);
                load_row<T, THREADS, NV>(a.error + (row + step) * a.cols, a.cols, t, err);
            }
            mean = mean_next; rstd = rstd_next;
        }
    }
    if (!a.partial) return;
    // the block's share: one row of dgain and one of dbias
    T* const out = a.partial + (int64_t)blockIdx.x * a.cols;
    const int64_t second = (int64_t)gridDim.x * a.cols;
    if constexpr (GROUPS == 1) {
        store_row<T, THREADS, NV>(out, a.cols, t, dgain);
        store_row<T, THREADS, NV>(out + second, a.cols, t, dbias);
    } else {
#pragma unroll
        for (int which = 0; which < 2; which++) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int e = 0; e < N; e++) share[group][(v * THREADS + t) * N + e] = which ? dbias[v][e] : dgain[v][e];
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += BLOCK) {
                T sum = share[0][c];
#pragma unroll
                for (int g = 1; g < GROUPS; g++) sum += share[g][c];
                out[which * second + c] = sum;
            }
        }
    }
}

// ---- rows that fit no block's registers ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(1024) void norm_forward_long_kernel(const NormArgs<T> a) {
    __shared__ T scratch[2][16];
    const T count = T(a.cols);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = a.src + row * a.pitch;
        T s[1] = {T(0)};
        for (int c = threadIdx.x; c < a.cols; c += 1024) s[0] += x[c];
        row_sums<T, 1024, 1>(s, scratch[0]);
        const T mean = s[0] / count;
        s[0] = T(0);
        for (int c = threadIdx.x; c < a.cols; c += 1024) { const T d = x[c] - mean; s[0] = mul_add(d, d, s[0]); }
        row_sums<T, 1024, 1>(s, scratch[1]);
        const T rstd = T(1) / root(s[0] / count + a.epsilon);
        for (int c = threadIdx.x; c < a.cols; c += 1024) a.drn[row * a.cols + c] = mul_add((x[c] - mean) * rstd, a.gain[c], a.bias[c]);
        if (threadIdx.x == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
    }
}
template <typename T>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const NormArgs<T> a) {
    __shared__ T scratch[2][2 * 16];
    const T count = T(a.cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const T *const x = a.src + row * a.pitch, *const err = a.error + row * a.cols;
        const T mean = a.mean[row], rstd = a.rstd[row];
        T s[2] = {T(0), T(0)};
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const T g = err[c] * a.gain[c];
            s[0] += g;
            s[1] = mul_add(g, (x[c] - mean) * rstd, s[1]);
        }
        row_sums<T, 1024, 2>(s, scratch[turn]);
        const T g_mean = s[0] / count, gh_mean = s[1] / count;
        for (int c = threadIdx.x; c < a.cols; c += 1024)
            a.d_src[row * a.cols + c] = rstd * (err[c] * a.gain[c] - mul_add((x[c] - mean) * rstd, gh_mean, g_mean));
    }
}
// blockIdx.y-th strip of rows, 256 columns per block
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const NormArgs<T> a, int64_t strip) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    const int64_t first = blockIdx.y * strip, last = first + strip < a.rows ? first + strip : a.rows;
    T dgain = T(0), dbias = T(0);
    for (int64_t row = first; row < last; row++) {
        const T e = a.error[row * a.cols + c];
        dgain = mul_add(e, (a.src[row * a.pitch + c] - a.mean[row]) * a.rstd[row], dgain);
        dbias += e;
    }
    a.partial[(int64_t)blockIdx.y * a.cols + c] = dgain;
    a.partial[((int64_t)gridDim.y + blockIdx.y) * a.cols + c] = dbias;
}

// Adds `parts` rows of shares: 16 wavefronts of a block take every 16th row of 64 columns, then their sums are added in order.
template <typename T>
__global__ __launch_bounds__(1024) void norm_add_shares_kernel(const T* __restrict__ partial, int parts, int cols, T* d_gain, T* d_bias) {
    __shared__ T sums[16][64];
    T* const out = blockIdx.y ? d_bias : d_gain;
    if (!out) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const T* const in = partial + (int64_t)blockIdx.y * parts * cols;
    T sum = T(0);
    if (c < cols) {
#pragma unroll 8
        for (int p = wave; p < parts; p += 16) sum += in[(int64_t)p * cols + c];
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < cols) {
        for (int w = 1; w < 16; w++) sum += sums[w][lane];
        out[c] = sum;
    }
}

// ---- plans ----------------------------------------------------------------------------------------------------------
// Calls `f.template operator()<BLOCK, THREADS, NV>()` for the narrowest of the groups of threads, a wavefront or a block, that holds a row; false: none does.
template <typename T, typename F>
static bool with_row_plan(int64_t cols, const F& f) {
    const int64_t vecs = (cols + Wide<T>::N - 1) / Wide<T>::N;
    if      (vecs <= 64)       f(std::integral_constant<int, 256>(), std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    else if (vecs <= 128)      f(std::integral_constant<int, 256>(), std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    else if (vecs <= 256)      f(std::integral_constant<int, 256>(), std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
    else if (vecs <= 512)      f(std::integral_constant<int, 256>(), std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    else if (vecs <= 1024)     f(std::integral_constant<int, 256>(), std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
    else if (vecs <= 2048)     f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
    else if (vecs <= 4096)     f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
    else return false;
    return true;
}

template <typename T>
static int forward(Device* dev, const NormArgs<T>& a) {
    const int64_t cus = dev->props.multiProcessorCount;
    const bool held = with_row_plan<T>(a.cols, [&](auto block, auto threads, auto nv) {
        constexpr int BLOCK = decltype(block)::value, THREADS = decltype(threads)::value, NV = decltype(nv)::value, GROUPS = BLOCK / THREADS;
        // blocks that stay and walk over the rows: with four vectors a thread 1024 threads per unit (4096 x 4096 floats 26.1 us, 2048 threads
        // 27.6), with fewer 2048 (2047 x 1111 8.4, 1024 threads 8.8)
        const int64_t all = (a.rows + GROUPS - 1) / GROUPS, most = cus * ((NV < 4 ? 2048 : 1024) / BLOCK);
        hipLaunchKernelGGL((norm_forward_kernel<T, BLOCK, THREADS, NV>), dim3((unsigned)(all < most ? all : most)), dim3(BLOCK), 0, dev->stream, a);
    });
    if (!held) hipLaunchKernelGGL((norm_forward_long_kernel<T>), dim3((unsigned)(a.rows < 2 * cus ? a.rows : 2 * cus)), dim3(1024), 0, dev->stream, a);
    NK_HIP(hipGetLastError());
    set_path(held ? "norm_rows" : "norm_long_rows");
    return NK_OK;
}

template <typename T>
static int backward(Device* dev, NormArgs<T> a, T* d_gain, T* d_bias) {
    const int64_t cus = dev->props.multiProcessorCount;
    const bool shares = d_gain || d_bias;
    int parts = 0, failed = NK_OK;
    const auto take = [&](int64_t n) {
        parts = (int)n;
        void* ws = nullptr;
        if (shares && !(failed = workspace(dev, (uint64_t)2 * n * a.cols * sizeof(T), &ws))) a.partial = (T*)ws;
        return failed == NK_OK;
    };
    const bool held = with_row_plan<T>(a.cols, [&](auto block, auto threads, auto nv) {
        constexpr int BLOCK = decltype(block)::value, THREADS = decltype(threads)::value, NV = decltype(nv)::value, GROUPS = BLOCK / THREADS;
        const int64_t all = (a.rows + GROUPS - 1) / GROUPS, most = cus * (BLOCK == 256 ? 2 : 1);
        if (!take(all < most ? all : most)) return;
        hipLaunchKernelGGL((norm_backward_kernel<T, BLOCK, THREADS, NV>), dim3((unsigned)parts), dim3(BLOCK), 0, dev->stream, a);
    });
    if (!held) {
        if (a.d_src)
            hipLaunchKernelGGL((norm_backward_long_kernel<T>), dim3((unsigned)(a.rows < 2 * cus ? a.rows : 2 * cus)), dim3(1024), 0, dev->stream, a);
        if (shares) {
            const int64_t strip = (a.rows + 63) / 64;
            if (take((a.rows + strip - 1) / strip))
                hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((unsigned)((a.cols + 255) / 256), (unsigned)parts), dim3(256), 0, dev->stream, a, strip);
        }
    }
    if (failed) return failed;
    if (shares)
        hipLaunchKernelGGL((norm_add_shares_kernel<T>), dim3((unsigned)((a.cols + 63) / 64), 2), dim3(1024), 0, dev->stream, (const T*)a.partial, parts, a.cols, d_gain, d_bias);
    NK_HIP(hipGetLastError());
    set_path(held ? "norm_rows_backward" : "norm_long_rows_backward");
    return NK_OK;
}

// Whether [a, a + n) and [b, b + m) share a byte.
static bool overlap(nk_buf a, uint64_t n, nk_buf b, uint64_t m) { return a && b && a < b + m && b < a + n; }

static int check_rows(const char* what, int dtype, int64_t rows, int64_t cols, int64_t pitch) {
    NK_REQUIRE(dtype == NK_F32 || dtype == NK_F64, "%s: unknown dtype %d", what, dtype);
    NK_REQUIRE(rows >= 1 && cols >= 1, "%s: rows and columns must be positive (got %lld, %lld)", what, (long long)rows, (long long)cols);
    // (norm_add_shares_kernel's 16 threads per column stay below the 2^32 of a launch)
    NK_REQUIRE(cols <= ((int64_t)1 << 27) - 1024, "%s: rows of %lld elements, 2^27-1024 are the most", what, (long long)cols);
    NK_REQUIRE(rows < ((int64_t)1 << 31) && rows * cols < ((int64_t)1 << 31), "%s: %lld x %lld exceeds 2^31-1 elements", what, (long long)rows, (long long)cols);
    NK_REQUIRE(pitch >= cols && pitch < ((int64_t)1 << 31), "%s: a pitch of %lld elements does not hold rows of %lld", what, (long long)pitch, (long long)cols);
    return NK_OK;
}

}  // namespace nk

using namespace nk;

extern "C" int nk_layer_norm(nk_dev h, int dtype, int64_t rows, int64_t cols, nk_buf src, int64_t src_pitch, nk_buf gain, nk_buf bias,
                             double epsilon, nk_buf drn, nk_buf mean, nk_buf rstd) {
    NK_DEVICE(dev, h);
    const char* what = "nk_layer_norm";
    if (int e = check_rows(what, dtype, rows, cols, src_pitch)) return e;
    NK_REQUIRE(epsilon >= 0 && epsilon < INFINITY, "%s: epsilon must be finite and not negative", what);
    NK_REQUIRE((mean == 0) == (rstd == 0), "%s: mean and rstd are kept together or not at all", what);
    const uint64_t eb = dtype_bytes(dtype), size = (uint64_t)(rows * cols) * eb, src_size = ((uint64_t)(rows - 1) * src_pitch + cols) * eb;
    if (int e = check_range(dev, "nk_layer_norm(src)", src, 0, src_size)) return e;
    if (int e = check_range(dev, "nk_layer_norm(gain)", gain, 0, cols * eb)) return e;
    if (int e = check_range(dev, "nk_layer_norm(bias)", bias, 0, cols * eb)) return e;
    if (int e = check_range(dev, "nk_layer_norm(drn)", drn, 0, size)) return e;
    if (mean) {
        if (int e = check_range(dev, "nk_layer_norm(mean)", mean, 0, rows * eb)) return e;
        if (int e = check_range(dev, "nk_layer_norm(rstd)", rstd, 0, rows * eb)) return e;
    }
    for (nk_buf b : {src, gain, bias, drn, mean, rstd}) NK_REQUIRE(b % eb == 0, "%s: a buffer does not start at an element", what);
    const nk_buf outs[3] = {drn, mean, rstd};
    const uint64_t lens[3] = {size, rows * eb, rows * eb};
    for (int i = 0; i < 3; i++) {
        const bool in_place = i == 0 && src == drn && src_pitch == cols;
        NK_REQUIRE((in_place || !overlap(outs[i], lens[i], src, src_size)) && !overlap(outs[i], lens[i], gain, cols * eb) && !overlap(outs[i], lens[i], bias, cols * eb),
                   "%s: an output overlaps an input", what);
        for (int j = 0; j < i; j++) NK_REQUIRE(!overlap(outs[i], lens[i], outs[j], lens[j]), "%s: two outputs overlap", what);
    }
    const auto run = [&](auto one) {
        typedef decltype(one) T;
        NormArgs<T> a{};
        a.src = (const T*)src; a.pitch = src_pitch; a.rows = rows; a.cols = (int)cols; a.gain = (const T*)gain; a.bias = (const T*)bias;
        a.epsilon = (T)epsilon; a.drn = (T*)drn; a.mean = (T*)mean; a.rstd = (T*)rstd;
        return forward<T>(dev, a);
    };
    return dtype == NK_F32 ? run(float()) : run(double());
}

extern "C" int nk_layer_norm_backward(nk_dev h, int dtype, int64_t rows, int64_t cols, nk_buf src, int64_t src_pitch, nk_buf gain, nk_buf mean,
                                      nk_buf rstd, nk_buf error, nk_buf d_src, nk_buf d_gain, nk_buf d_bias) {
    NK_DEVICE(dev, h);
    const char* what = "nk_layer_norm_backward";
    if (int e = check_rows(what, dtype, rows, cols, src_pitch)) return e;
    NK_REQUIRE(d_src || d_gain || d_bias, "%s: no gradient is asked for", what);
    const uint64_t eb = dtype_bytes(dtype), size = (uint64_t)(rows * cols) * eb, src_size = ((uint64_t)(rows - 1) * src_pitch + cols) * eb;
    const nk_buf ins[5] = {src, gain, mean, rstd, error}, outs[3] = {d_src, d_gain, d_bias};
    const uint64_t in_lens[5] = {src_size, cols * eb, rows * eb, rows * eb, size}, out_lens[3] = {size, cols * eb, cols * eb};
    const char* const in_names[5] = {"nk_layer_norm_backward(src)", "nk_layer_norm_backward(gain)", "nk_layer_norm_backward(mean)",
                                     "nk_layer_norm_backward(rstd)", "nk_layer_norm_backward(error)"};
    const char* const out_names[3] = {"nk_layer_norm_backward(d_src)", "nk_layer_norm_backward(d_gain)", "nk_layer_norm_backward(d_bias)"};
    for (nk_buf b : {src, gain, mean, rstd, error, d_src, d_gain, d_bias}) NK_REQUIRE(b % eb == 0, "%s: a buffer does not start at an element", what);
    for (int i = 0; i < 5; i++)
        if (int e = check_range(dev, in_names[i], ins[i], 0, in_lens[i])) return e;
    for (int i = 0; i < 3; i++) {
        if (!outs[i]) continue;
        if (int e = check_range(dev, out_names[i], outs[i], 0, out_lens[i])) return e;
        for (int j = 0; j < 5; j++) NK_REQUIRE(!overlap(outs[i], out_lens[i], ins[j], in_lens[j]), "%s: a gradient overlaps an input", what);
        for (int j = 0; j < i; j++) NK_REQUIRE(!overlap(outs[i], out_lens[i], outs[j], out_lens[j]), "%s: two gradients overlap", what);
    }
    const auto run = [&](auto one) {
        typedef decltype(one) T;
        NormArgs<T> a{};
        a.src = (const T*)src; a.pitch = src_pitch; a.rows = rows; a.cols = (int)cols; a.gain = (const T*)gain;
        a.mean = (T*)mean; a.rstd = (T*)rstd; a.error = (const T*)error; a.d_src = (T*)d_src;
        return backward<T>(dev, a, (T*)d_gain, (T*)d_bias);
    };
    return dtype == NK_F32 ? run(float()) : run(double());
}
