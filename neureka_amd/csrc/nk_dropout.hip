// nk_dropout: y = keep ? x / (1 - p) : 0, keep drawn by a counter-based generator.
//
// Element i (row-major index) belongs to word i % 4 of the block i / 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw:
// "Parallel random numbers: as easy as 1, 2, 3", 2011) with key = seed and counter = (i / 4, offset); it is kept where the word is at
// least floor(p 2^32).  Nothing is stored: the same seed and offset give the same mask again, so the backward pass is the same call on
// the error.  A thread makes one block of the generator and moves the four elements that belong to it; the ten rounds (20
// 32 x 32 -> 64-bit products, 60 further integer operations) run beside the memory traffic, which bounds the kernel: x in, y out
// (4096 x 4096 floats 24 us, 5.6 TB/s).
#include "nk_internal.h"
#include "nk_views.h"

namespace nk {

struct Mask { uint32_t key0, key1, offset0, offset1; uint64_t threshold; };     // threshold up to 2^32: everything dropped

__device__ __forceinline__ void philox(uint64_t block, const Mask& m, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = m.offset0, c3 = m.offset1, k0 = m.key0, k1 = m.key1;
#pragma unroll
    for (int round = 0; round < 10; round++) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0; c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1; c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// dense source and drain, starting at any element
template <typename T>
__global__ __launch_bounds__(256) void dropout_dense_kernel(const T* src, T* drn, int64_t n, const Mask m, T scale) {
    typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = block * 4;
    if (i >= n) return;
    uint32_t w[4];
    if (i + 4 <= n) {
        V x = *(const V*)(src + i);
        philox((uint64_t)block, m, w);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = w[e] >= m.threshold ? x[e] * scale : T(0);
        *(V*)(drn + i) = x;
    } else {
        philox((uint64_t)block, m, w);
        for (int e = 0; i + e < n; e++) drn[i + e] = w[e] >= m.threshold ? src[i + e] * scale : T(0);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void dropout_view_kernel(const T* src, const Cfg src_cfg, T* drn, const Cfg drn_cfg, int rank, int64_t n, const Mask m, T scale) {
    const int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = block * 4;
    if (i >= n) return;
    uint32_t w[4];
    philox((uint64_t)block, m, w);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (i + e >= n) break;
        int idx[NK_MAX_RANK];
        nd_of_flat(drn_cfg, rank, (int)(i + e), idx);
        const T x = src[phys_of_nd(src_cfg, rank, idx)];
        drn[phys_of_nd(drn_cfg, rank, idx)] = w[e] >= m.threshold ? x * scale : T(0);
    }
}

template <typename T>
static int dropout(Device* dev, int rank, nk_buf drn, Cfg& dc, nk_buf src, Cfg& sc, const Mask& m, double scale, int64_t n) {
    const unsigned grid = (unsigned)(((n + 3) / 4 + 255) / 256);
    const Cfg* cfgs[2] = {&dc, &sc};
    const bool own[2] = {false, false};                     // both are addressed with the drain's nd-index
    Canon c;
    const bool simple = canonicalize(c, rank, dc.shape, 2, cfgs, nullptr, own);
    if (simple && (c.rank == 0 || (c.rank == 1 && c.stride[0][0] == 1 && c.stride[1][0] == 1))) {
        hipLaunchKernelGGL((dropout_dense_kernel<T>), dim3(grid), dim3(256), 0, dev->stream, (const T*)src + c.base[1], (T*)drn + c.base[0], n, m, (T)scale);
        set_path("dropout_dense");
    } else {
        hipLaunchKernelGGL((dropout_view_kernel<T>), dim3(grid), dim3(256), 0, dev->stream, (const T*)src, sc, (T*)drn, dc, rank, n, m, (T)scale);
        set_path("dropout_view");
    }
    NK_HIP(hipGetLastError());
    return NK_OK;
}

}  // namespace nk

using namespace nk;

extern "C" int nk_dropout(nk_dev h, int dtype, int rank, nk_buf drn, const int32_t* drn_cfg, nk_buf src, const int32_t* src_cfg,
                          double probability, uint64_t seed, uint64_t offset, int64_t n) {
    NK_DEVICE(dev, h);
    NK_REQUIRE(dtype == NK_F32 || dtype == NK_F64, "nk_dropout: unknown dtype %d", dtype);
    if (int e = check_cfg("nk_dropout(drn)", drn_cfg, rank)) return e;
    if (int e = check_cfg("nk_dropout(src)", src_cfg, rank)) return e;
    NK_REQUIRE(probability >= 0 && probability <= 1, "nk_dropout: the probability of a drop must lie in [0, 1]");
    int64_t size = 1;
    for (int k = 0; k < rank; k++) {
        NK_REQUIRE(drn_cfg[k] == src_cfg[k], "nk_dropout: source and drain differ in axis %d (%d and %d)", k, src_cfg[k], drn_cfg[k]);
        size *= drn_cfg[k];
        NK_REQUIRE(size < ((int64_t)1 << 31), "nk_dropout: more than 2^31-1 elements");
    }
    NK_REQUIRE(n == size, "nk_dropout: n = %lld, the drain has %lld elements", (long long)n, (long long)size);
    const int eb = dtype_bytes(dtype);
    NK_REQUIRE(drn % eb == 0 && src % eb == 0, "nk_dropout: a buffer does not start at an element");
    if (int e = check_extent(dev, "nk_dropout(drn)", drn, drn_cfg, rank, eb)) return e;
    if (int e = check_extent(dev, "nk_dropout(src)", src, src_cfg, rank, eb)) return e;
    Cfg dc, sc;
    load_cfg(dc, drn_cfg, rank);
    load_cfg(sc, src_cfg, rank);
    const auto view_of = [&](nk_buf at, const Cfg& c) {
        View v;
        v.first = (int64_t)(at / eb);
        v.rank = rank;
        for (int k = 0; k < rank; k++) {
            v.first += (int64_t)c.offset[k] * c.strides[k];
            v.extent[k] = c.shape[k];
            v.step[k] = (int64_t)c.strides[k] * c.spread[k];
        }
        return v;
    };
    static_assert(View::MOST == NK_MAX_RANK, "a view has as many axes as a descriptor");
    const View to = view_of(drn, dc), from = view_of(src, sc);
    bool in_place = to.first == from.first;                 // (every element is read and written by the same thread)
    for (int k = 0; k < rank; k++) {
        NK_REQUIRE(to.extent[k] == 1 || to.step[k] != 0, "nk_dropout: axis %d of the drain holds one element %lld times", k, (long long)to.extent[k]);
        in_place = in_place && (to.extent[k] == 1 || to.step[k] == from.step[k]);
    }
    NK_REQUIRE(in_place || !views_meet(to, from), "nk_dropout: the drain overlaps the source without being the same view of it");
    int64_t prod = 1;                                       // the mask follows the row-major index whatever table a view carries
    for (int k = rank - 1; k >= 0; k--) { dc.imap[k] = (int)prod; prod *= dc.shape[k]; }
    const Mask m = {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32), (uint64_t)(probability * 4294967296.0)};
    const double scale = probability < 1 ? 1.0 / (1.0 - probability) : 0.0;
    return dtype == NK_F32 ? dropout<float>(dev, rank, drn, dc, src, sc, m, scale, n) : dropout<double>(dev, rank, drn, dc, src, sc, m, scale, n);
}
