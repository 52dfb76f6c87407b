// layer_norm.cu -- layer norm with its residual add, forward and backward (C ABI
// morpho_sm100_layer_norm_*).  Per row of `dim` values
//   h = x + residual (rounded to their type and stored; h = x without a residual)
//   mu = mean(h),  var = mean((h - mu)^2),  r = 1 / sqrt(var + eps),  xh = (h - mu) r
//   y = xh * weight + bias
// and, with g = dy * weight,
//   dx = r (g - mean(g) - xh mean(g xh)) + dh,   dweight = sum_rows dy xh,   dbias = sum_rows dy
// where dh is the gradient that reaches h directly (the residual stream).
//
// The work per element is a few operations, so HBM bounds it: every tensor is read once and written
// once.  The variance is the second moment about the mean just formed, which loses nothing to
// cancellation.  All sums are fp32.
//
// Many rows (the *_stream kernels): a persistent CTA of eight warps, 1 to 8 of them to a row, a lane holding
// up to 32 of its elements.  Each group of warps keeps a ring of rows in flight as bulk copies into shared
// memory, so the bytes in flight do not depend on registers or occupancy, which the backward's dweight /
// dbias sums (two fp32 registers per column, kept over all rows of the group) would otherwise limit.  The
// CTA's groups join their sums in a fixed order and write one fp32 partial row per CTA; a second kernel
// sums those in a fixed order (no atomics: the same bits every run).
// Few rows, or rows that are not 16-byte aligned: a warp or a CTA loads its row into registers.  Rows longer
// than a CTA's registers hold (dim > 8192) are read again from L2.
#include <algorithm>

#include "elem.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace morpho {
namespace {

constexpr int kCta = 256;        // threads per row of the CTA-wide kernels
constexpr int kWarpsPerCta = 4;  // rows at a time of the warp-wide kernels
constexpr int kMaxRegElems = 32; // row elements a thread holds

constexpr uint32_t K_NORM = 7;   // kernel id in the device status word

struct NormArgs {
    int64_t rows;
    int dim, wtype;
    float eps;
    int64_t sx, sres, sgy, sgh;  // row strides in elements
    const void *x, *res, *w, *b; // forward inputs (x is h in the backward)
    void *y, *h;
    float *mean, *rstd;
    const void *gy, *gh;
    void* dx;
    float* part;  // [grid][2][dim] partial dweight / dbias
    uint32_t* status;
    int stages;   // rows in flight per group of the streaming kernels
};

// Sum of two values over the group; every thread gets the result.  GROUP 256 uses `scratch` (16
// float2, used alternately by `turn`, so that one barrier per call suffices).
template <int GROUP>
__device__ __forceinline__ float2 group_sum(float a, float b, float2* scratch, int turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (GROUP == 32) return make_float2(a, b);
    const int warp = threadIdx.x >> 5;
    float2* s = scratch + (turn & 1) * 8;
    if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
    __syncthreads();
    float2 r = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r.x += s[i].x;
        r.y += s[i].y;
    }
    return r;
}

// NV packs of VEC elements per thread: pack i of thread l starts at column (i * GROUP + l) * VEC.
template <class T, int VEC, int NV, int GROUP>
__global__ void __launch_bounds__(GROUP == 32 ? 32 * kWarpsPerCta : kCta) layer_norm_fwd_kernel(const NormArgs a) {
    __shared__ float2 scratch[16];
    const int l = GROUP == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = GROUP == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;  // a whole warp, or never (GROUP 256)
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    float v[NV * VEC];
    Pack<T, VEC> px[NV], pr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * GROUP + l) * VEC;
        if (c < a.dim) px[i] = load_pack<T, VEC>(x + c);
    }
    if (a.res != nullptr) {
        const T* res = static_cast<const T*>(a.res) + row * a.sres;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * GROUP + l) * VEC;
            if (c < a.dim) pr[i] = load_pack<T, VEC>(res + c);
        }
        T* h = static_cast<T*>(a.h) + row * a.dim;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * GROUP + l) * VEC;
            if (c >= a.dim) continue;
#pragma unroll
            for (int k = 0; k < VEC; ++k) px[i].v[k] = from_f32<T>(to_f32(px[i].v[k]) + to_f32(pr[i].v[k]));
            store_pack<T, VEC>(h + c, px[i]);
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            v[i * VEC + k] = (i * GROUP + l) * VEC < a.dim ? to_f32(px[i].v[k]) : 0.f;
            sum += v[i * VEC + k];
        }
    const float inv = 1.0f / static_cast<float>(a.dim);
    const float mu = group_sum<GROUP>(sum, 0.f, scratch, 0).x * inv;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            v[i * VEC + k] -= mu;
            if ((i * GROUP + l) * VEC < a.dim) sq = fmaf(v[i * VEC + k], v[i * VEC + k], sq);
        }
    const float r = rsqrtf(group_sum<GROUP>(sq, 0.f, scratch, 1).x * inv + a.eps);
    if (l == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
    }
    T* y = static_cast<T*>(a.y) + row * a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * GROUP + l) * VEC;
        if (c >= a.dim) continue;
        Pack<T, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float w = a.w != nullptr ? load_as_f32(a.w, a.wtype, c + k) : 1.f;
            const float b = a.b != nullptr ? load_as_f32(a.b, a.wtype, c + k) : 0.f;
            o.v[k] = from_f32<T>(fmaf(v[i * VEC + k] * r, w, b));
        }
        store_pack<T, VEC>(y + c, o);
    }
}

// Any dim: one CTA per row, the row read three times (from L2 after the first).
template <class T>
__global__ void __launch_bounds__(kCta) layer_norm_fwd_long_kernel(const NormArgs a) {
    __shared__ float2 scratch[16];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    const T* res = a.res != nullptr ? static_cast<const T*>(a.res) + row * a.sres : nullptr;
    T* h = res != nullptr ? static_cast<T*>(a.h) + row * a.dim : nullptr;
    float sum = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += kCta) {
        T e = x[c];
        if (res != nullptr) {
            e = from_f32<T>(to_f32(e) + to_f32(res[c]));
            h[c] = e;  // read again by this thread only
        }
        sum += to_f32(e);
    }
    const T* src = res != nullptr ? h : x;
    const float inv = 1.0f / static_cast<float>(a.dim);
    const float mu = group_sum<kCta>(sum, 0.f, scratch, 0).x * inv;
    float sq = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += kCta) {
        const float d = to_f32(src[c]) - mu;
        sq = fmaf(d, d, sq);
    }
    const float r = rsqrtf(group_sum<kCta>(sq, 0.f, scratch, 1).x * inv + a.eps);
    if (threadIdx.x == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
    }
    T* y = static_cast<T*>(a.y) + row * a.dim;
    for (int c = threadIdx.x; c < a.dim; c += kCta) {
        const float w = a.w != nullptr ? load_as_f32(a.w, a.wtype, c) : 1.f;
        const float b = a.b != nullptr ? load_as_f32(a.b, a.wtype, c) : 0.f;
        y[c] = from_f32<T>(fmaf((to_f32(src[c]) - mu) * r, w, b));
    }
}

template <class T, int VEC, int NV, int GROUP>
__global__ void __launch_bounds__(GROUP == 32 ? 32 * kWarpsPerCta : kCta) layer_norm_bwd_kernel(const NormArgs a) {
    constexpr int E = NV * VEC;
    __shared__ float2 scratch[16];
    const int l = GROUP == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t first = GROUP == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (GROUP == 32 ? kWarpsPerCta : 1);
    float dw[E], db[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    const float inv = 1.0f / static_cast<float>(a.dim);
    int turn = 0;
    for (int64_t row = first; row < a.rows; row += step, ++turn) {
        const T* h = static_cast<const T*>(a.x) + row * a.sx;
        const T* gy = static_cast<const T*>(a.gy) + row * a.sgy;
        const float mu = a.mean[row], r = a.rstd[row];
        Pack<T, VEC> ph[NV], pg[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * GROUP + l) * VEC;
            if (c < a.dim) {
                ph[i] = load_pack<T, VEC>(h + c);
                pg[i] = load_pack<T, VEC>(gy + c);
            }
        }
        float s0 = 0.f, s1 = 0.f;
        float xh[E], g[E];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * GROUP + l) * VEC;
            if (c < a.dim) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    const float d = to_f32(pg[i].v[k]);
                    xh[e] = (to_f32(ph[i].v[k]) - mu) * r;
                    dw[e] = fmaf(d, xh[e], dw[e]);
                    db[e] += d;
                    g[e] = a.w != nullptr ? d * load_as_f32(a.w, a.wtype, c + k) : d;
                    s0 += g[e];
                    s1 = fmaf(g[e], xh[e], s1);
                }
            }
        }
        const float2 s = group_sum<GROUP>(s0, s1, scratch, turn);
        const float mg = s.x * inv, mgx = s.y * inv;
        T* dx = static_cast<T*>(a.dx) + row * a.dim;
        const T* gh = a.gh != nullptr ? static_cast<const T*>(a.gh) + row * a.sgh : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * GROUP + l) * VEC;
            if (c >= a.dim) continue;
            Pack<T, VEC> o, pd;
            if (gh != nullptr) pd = load_pack<T, VEC>(gh + c);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const int e = i * VEC + k;
                float d = r * (g[e] - mg - xh[e] * mgx);
                if (gh != nullptr) d += to_f32(pd.v[k]);
                o.v[k] = from_f32<T>(d);
            }
            store_pack<T, VEC>(dx + c, o);
        }
    }
    if (a.part == nullptr) return;
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
    if (GROUP == 32) {
        // the CTA's warps add their sums in turn (shared memory: one dweight and one dbias row)
        extern __shared__ float rows[];
        for (int w = 0; w < kWarpsPerCta; ++w) {
            if ((threadIdx.x >> 5) == w) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        const int c = (i * GROUP + l) * VEC + k;
                        if (c >= a.dim) continue;
                        rows[c] = w == 0 ? dw[i * VEC + k] : rows[c] + dw[i * VEC + k];
                        rows[a.dim + c] = w == 0 ? db[i * VEC + k] : rows[a.dim + c] + db[i * VEC + k];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * a.dim; c += 32 * kWarpsPerCta) part[c] = rows[c];
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const int c = (i * GROUP + l) * VEC + k;
                if (c >= a.dim) continue;
                part[c] = dw[i * VEC + k];
                part[a.dim + c] = db[i * VEC + k];
            }
    }
}

// Any dim: dx alone, one CTA per row, the row read twice.
template <class T>
__global__ void __launch_bounds__(kCta) layer_norm_bwd_long_kernel(const NormArgs a) {
    __shared__ float2 scratch[16];
    const int64_t row = blockIdx.x;
    const T* h = static_cast<const T*>(a.x) + row * a.sx;
    const T* gy = static_cast<const T*>(a.gy) + row * a.sgy;
    const T* gh = a.gh != nullptr ? static_cast<const T*>(a.gh) + row * a.sgh : nullptr;
    const float mu = a.mean[row], r = a.rstd[row];
    float s0 = 0.f, s1 = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += kCta) {
        const float g = to_f32(gy[c]) * (a.w != nullptr ? load_as_f32(a.w, a.wtype, c) : 1.f);
        s0 += g;
        s1 = fmaf(g, (to_f32(h[c]) - mu) * r, s1);
    }
    const float2 s = group_sum<kCta>(s0, s1, scratch, 0);
    const float inv = 1.0f / static_cast<float>(a.dim);
    const float mg = s.x * inv, mgx = s.y * inv;
    T* dx = static_cast<T*>(a.dx) + row * a.dim;
    for (int c = threadIdx.x; c < a.dim; c += kCta) {
        const float g = to_f32(gy[c]) * (a.w != nullptr ? load_as_f32(a.w, a.wtype, c) : 1.f);
        float d = r * (g - mg - (to_f32(h[c]) - mu) * r * mgx);
        if (gh != nullptr) d += to_f32(gh[c]);
        dx[c] = from_f32<T>(d);
    }
}

// Any dim: the weight and bias sums of one block of rows per blockIdx.y, a thread per column.
template <class T>
__global__ void __launch_bounds__(kCta) layer_norm_bwd_cols_kernel(const NormArgs a, int64_t rows_per_block) {
    const int c = blockIdx.x * kCta + threadIdx.x;
    if (c >= a.dim) return;
    const int64_t r0 = blockIdx.y * rows_per_block;
    const int64_t r1 = min(a.rows, r0 + rows_per_block);
    float dw = 0.f, db = 0.f;
    for (int64_t row = r0; row < r1; ++row) {
        const float d = to_f32(static_cast<const T*>(a.gy)[row * a.sgy + c]);
        const float xh = (to_f32(static_cast<const T*>(a.x)[row * a.sx + c]) - a.mean[row]) * a.rstd[row];
        dw = fmaf(d, xh, dw);
        db += d;
    }
    float* part = a.part + static_cast<int64_t>(blockIdx.y) * 2 * a.dim;
    part[c] = dw;
    part[a.dim + c] = db;
}

// ---- streaming kernels: aligned rows, up to 32 elements a lane ---------------------------------------

constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = 32 * kStreamWarps;
constexpr int kMaxStages = 8;

// Sums of two values over the W warps of a group (threads 32 W of the CTA, group `g`).
template <int W>
__device__ __forceinline__ float2 warps_sum(float a, float b, float2 (*scratch)[kStreamWarps], int turn, int g) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (W == 1) return make_float2(a, b);
    float2* s = scratch[turn & 1] + g * W;
    if ((threadIdx.x & 31) == 0) s[(threadIdx.x >> 5) & (W - 1)] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(1 + g), "n"(32 * W) : "memory");
    float2 r = s[0];
#pragma unroll
    for (int i = 1; i < W; ++i) {
        r.x += s[i].x;
        r.y += s[i].y;
    }
    return r;
}

// The ring of one group: stage i holds one row of each of up to three tensors.
struct RowRing {
    uint32_t data, bars;  // shared-memory addresses
    uint32_t row_bytes, stage_bytes;
    int stages;

    // One thread: fetch row `row` of the given tensors (NULL: none) as use number i of the ring.
    __device__ void fetch(int i, const void* a, const void* b, const void* c) const {
        const int s = i % stages;
        const uint32_t bar = bars + 8 * s, dst = data + s * stage_bytes;
        mbar_arrive_expect_tx(bar, row_bytes * (1 + (b != nullptr) + (c != nullptr)));
        bulk_load(dst, a, row_bytes, bar);
        if (b != nullptr) bulk_load(dst + row_bytes, b, row_bytes, bar);
        if (c != nullptr) bulk_load(dst + 2 * row_bytes, c, row_bytes, bar);
    }
    // After a wait for use i ran out: the copies that may still be in flight, each waited for in turn.
    __device__ void drain(int i, uint32_t* status) const {
        for (int k = 1; k < stages; ++k) mbar_wait(bars + 8 * ((i + k) % stages), ((i + k) / stages) & 1, status, K_NORM, 3);
    }
    __device__ uint32_t stage(int i) const { return data + (i % stages) * stage_bytes; }
    __device__ bool wait(int i, uint32_t* status, uint32_t site) const {
        return mbar_wait(bars + 8 * (i % stages), (i / stages) & 1, status, K_NORM, site);
    }
};

template <class T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> shared_pack(uint32_t addr) {
    const uint4 x = ld_shared_u4(addr);
    return *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(&x);
}

// Barriers and rings of the CTA's groups; every thread calls it.  Shared memory: rings, one after the other.
template <int W>
__device__ __forceinline__ RowRing make_ring(uint8_t* smem, uint64_t* bars, const NormArgs& a, int row_bytes, int tensors) {
    const int g = threadIdx.x / (32 * W);
    RowRing r;
    r.row_bytes = row_bytes;
    r.stage_bytes = row_bytes * tensors;
    r.stages = a.stages;
    r.data = smem_u32(smem) + g * a.stages * r.stage_bytes;
    r.bars = smem_u32(bars + g * kMaxStages);
    if (threadIdx.x < kStreamWarps / W * kMaxStages) mbar_init(smem_u32(bars + threadIdx.x), 1);
    fence_barrier_init();
    __syncthreads();
    return r;
}

template <class T, int NV, int W>
__global__ void __launch_bounds__(kStreamThreads, 2) layer_norm_fwd_stream_kernel(const NormArgs a) {
    constexpr int VEC = 16 / sizeof(T), E = NV * VEC, G = 32 * W, GROUPS = kStreamWarps / W;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[GROUPS * kMaxStages];
    __shared__ float2 scratch[2][kStreamWarps];
    pdl_release();
    const int l = threadIdx.x % G, g = threadIdx.x / G;
    const RowRing ring = make_ring<W>(smem, bars, a, a.dim * static_cast<int>(sizeof(T)), a.res != nullptr ? 2 : 1);
    pdl_wait();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * GROUPS + g, step = static_cast<int64_t>(gridDim.x) * GROUPS;
    const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.res);
    auto fetch = [&](int i, int64_t row) {
        if (row < a.rows) ring.fetch(i, x + row * a.sx, res != nullptr ? res + row * a.sres : nullptr, nullptr);
    };
    if (l == 0)
        for (int i = 0; i < a.stages; ++i) fetch(i, first + i * step);
    float w[E], b[E];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int c = (i * G + l) * VEC + k;
            w[i * VEC + k] = a.w != nullptr && c < a.dim ? load_as_f32(a.w, a.wtype, c) : 1.f;
            b[i * VEC + k] = a.b != nullptr && c < a.dim ? load_as_f32(a.b, a.wtype, c) : 0.f;
        }
    const float inv = 1.0f / static_cast<float>(a.dim);
    int i = 0;
    for (int64_t row = first; row < a.rows; row += step, ++i) {
        if (!ring.wait(i, a.status, 1)) {
            ring.drain(i, a.status);
            break;
        }
        const uint32_t src = ring.stage(i);
        float v[E];
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + l) * VEC;
            if (c < a.dim) {
                Pack<T, VEC> p = shared_pack<T>(src + c * sizeof(T));
                if (res != nullptr) {
                    const Pack<T, VEC> q = shared_pack<T>(src + ring.row_bytes + c * sizeof(T));
#pragma unroll
                    for (int k = 0; k < VEC; ++k) p.v[k] = from_f32<T>(to_f32(p.v[k]) + to_f32(q.v[k]));
                    store_pack<T, VEC>(static_cast<T*>(a.h) + row * a.dim + c, p);
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v[n * VEC + k] = to_f32(p.v[k]);
                    sum += v[n * VEC + k];
                }
            }
        }
        const float mu = warps_sum<W>(sum, 0.f, scratch, 0, g).x * inv;
        __syncwarp();
        if (l == 0) fetch(i + a.stages, row + a.stages * step);  // the whole group has read the stage
        float sq = 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n)
            if ((n * G + l) * VEC < a.dim) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v[n * VEC + k] -= mu;
                    sq = fmaf(v[n * VEC + k], v[n * VEC + k], sq);
                }
            }
        const float r = rsqrtf(warps_sum<W>(sq, 0.f, scratch, 1, g).x * inv + a.eps);
        if (l == 0) {
            a.mean[row] = mu;
            a.rstd[row] = r;
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + l) * VEC;
            if (c < a.dim) {
                Pack<T, VEC> o;
#pragma unroll
                for (int k = 0; k < VEC; ++k) o.v[k] = from_f32<T>(fmaf(v[n * VEC + k] * r, w[n * VEC + k], b[n * VEC + k]));
                store_pack<T, VEC>(static_cast<T*>(a.y) + row * a.dim + c, o);
            }
        }
    }
}

template <class T, int NV, int W>
__global__ void __launch_bounds__(kStreamThreads, NV * 16 / sizeof(T) > 16 ? 1 : 2) layer_norm_bwd_stream_kernel(const NormArgs a) {
    constexpr int VEC = 16 / sizeof(T), E = NV * VEC, G = 32 * W, GROUPS = kStreamWarps / W;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[GROUPS * kMaxStages];
    __shared__ float2 scratch[2][kStreamWarps];
    pdl_release();
    const int l = threadIdx.x % G, g = threadIdx.x / G;
    const int tensors = a.gh != nullptr ? 3 : 2;
    const RowRing ring = make_ring<W>(smem, bars, a, a.dim * static_cast<int>(sizeof(T)), tensors);
    float* ws = reinterpret_cast<float*>(smem + GROUPS * a.stages * ring.stage_bytes);  // the weight, fp32
    pdl_wait();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * GROUPS + g, step = static_cast<int64_t>(gridDim.x) * GROUPS;
    const T *h = static_cast<const T*>(a.x), *gy = static_cast<const T*>(a.gy), *gh = static_cast<const T*>(a.gh);
    auto fetch = [&](int i, int64_t row) {
        if (row < a.rows) ring.fetch(i, h + row * a.sx, gy + row * a.sgy, gh != nullptr ? gh + row * a.sgh : nullptr);
    };
    if (l == 0)
        for (int i = 0; i < a.stages; ++i) fetch(i, first + i * step);
    for (int c = threadIdx.x; c < a.dim; c += kStreamThreads) ws[c] = a.w != nullptr ? load_as_f32(a.w, a.wtype, c) : 1.f;
    __syncthreads();
    float dw[E], db[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    const float inv = 1.0f / static_cast<float>(a.dim);
    int i = 0;
    float mu = 0.f, r = 0.f;
    if (first < a.rows) {
        mu = a.mean[first];
        r = a.rstd[first];
    }
    for (int64_t row = first; row < a.rows; row += step, ++i) {
        const int64_t next = row + step < a.rows ? row + step : row;
        const float mu1 = a.mean[next], r1 = a.rstd[next];  // in flight beside this row
        if (!ring.wait(i, a.status, 2)) {
            ring.drain(i, a.status);
            break;
        }
        const uint32_t src = ring.stage(i);
        float s0 = 0.f, s1 = 0.f;
        float xh[E], gw[E];
        Pack<T, VEC> ph[NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + l) * VEC;
            if (c < a.dim) {
                const Pack<T, VEC> p = shared_pack<T>(src + c * sizeof(T)), q = shared_pack<T>(src + ring.row_bytes + c * sizeof(T));
                if (gh != nullptr) ph[n] = shared_pack<T>(src + 2 * ring.row_bytes + c * sizeof(T));
                float w[VEC];
#pragma unroll
                for (int k = 0; k < VEC; k += 4) {
                    const float4 w4 = *reinterpret_cast<const float4*>(ws + c + k);
                    w[k] = w4.x, w[k + 1] = w4.y, w[k + 2] = w4.z, w[k + 3] = w4.w;
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = n * VEC + k;
                    const float d = to_f32(q.v[k]);
                    xh[e] = (to_f32(p.v[k]) - mu) * r;
                    dw[e] = fmaf(d, xh[e], dw[e]);
                    db[e] += d;
                    gw[e] = d * w[k];
                    s0 += gw[e];
                    s1 = fmaf(gw[e], xh[e], s1);
                }
            }
        }
        const float2 s = warps_sum<W>(s0, s1, scratch, i, g);
        __syncwarp();
        if (l == 0) fetch(i + a.stages, row + a.stages * step);
        const float mg = s.x * inv, mgx = s.y * inv;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + l) * VEC;
            if (c < a.dim) {
                Pack<T, VEC> o;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = n * VEC + k;
                    float d = r * (gw[e] - mg - xh[e] * mgx);
                    if (gh != nullptr) d += to_f32(ph[n].v[k]);
                    o.v[k] = from_f32<T>(d);
                }
                store_pack<T, VEC>(static_cast<T*>(a.dx) + row * a.dim + c, o);
            }
        }
        mu = mu1;
        r = r1;
    }
    if (a.part == nullptr) return;
    // the groups add their sums in turn, over the rings (every fetched row has been waited for)
    float* rows = reinterpret_cast<float*>(smem);
    __syncthreads();
    for (int t = 0; t < GROUPS; ++t) {
        if (g == t) {
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int c = (n * G + l) * VEC + k;
                    if (c < a.dim) {
                        rows[c] = t == 0 ? dw[n * VEC + k] : rows[c] + dw[n * VEC + k];
                        rows[a.dim + c] = t == 0 ? db[n * VEC + k] : rows[a.dim + c] + db[n * VEC + k];
                    }
                }
        }
        __syncthreads();
    }
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
    for (int c = threadIdx.x; c < 2 * a.dim; c += kStreamThreads) part[c] = rows[c];
}

// dweight / dbias = the sums of the `n` partial rows, in a fixed order: 32 columns per block, 32 threads a
// column.
__global__ void __launch_bounds__(1024) layer_norm_reduce_kernel(const float* part, int n, int dim, int wtype, void* dw, void* db) {
    __shared__ float s[32][33];
    pdl_release();
    pdl_wait();
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + cx, width = 2 * static_cast<int64_t>(dim);
    float sum = 0.f;
    if (c < width) {
#pragma unroll 4
        for (int i = ry; i < n; i += 32) sum += part[i * width + c];
    }
    s[ry][cx] = sum;
    __syncthreads();
    sum = s[cx][ry];  // one warp a column
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + ry;
    if (cx != 0 || col >= width) return;
    if (col < dim) {
        if (dw != nullptr) store_from_f32(dw, wtype, col, sum);
    } else if (db != nullptr) {
        store_from_f32(db, wtype, col - dim, sum);
    }
}

// ---- host ---------------------------------------------------------------------------------

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether every row of a tensor (base, row stride in elements) starts on a 16-byte boundary.
bool rows_aligned(const void* p, int64_t stride, int type) {
    return p == nullptr || (aligned16(p) && stride * dtype_bytes(type) % 16 == 0);
}

int validate_norm(const morpho_layer_norm_t* p) {
    if (p == nullptr) return set_error(MORPHO_ERR_INVALID, "layer norm problem is NULL");
    if (p->rows < 0 || p->rows > 2147483647LL) return set_error(MORPHO_ERR_INVALID, "layer norm: rows = %lld out of range", static_cast<long long>(p->rows));
    if (p->dim <= 0 || p->dim > (1 << 24)) return set_error(MORPHO_ERR_INVALID, "layer norm: dim = %d out of range", p->dim);
    if (p->type < MORPHO_DTYPE_F16 || p->type > MORPHO_DTYPE_F32)
        return set_error(MORPHO_ERR_INVALID, "layer norm: unknown element type %d", p->type);
    if (p->weight_type != p->type && p->weight_type != MORPHO_DTYPE_F32)
        return set_error(MORPHO_ERR_INVALID, "layer norm: weights must have the input's type or be fp32");
    if (!(p->eps >= 0.0f)) return set_error(MORPHO_ERR_INVALID, "layer norm: eps must be non-negative");
    for (const int64_t s : {p->stride_x, p->stride_residual, p->stride_grad_y, p->stride_grad_h})
        if (s != 0 && s < p->dim) return set_error(MORPHO_ERR_INVALID, "layer norm: row stride %lld below dim %d", static_cast<long long>(s), p->dim);
    return MORPHO_OK;
}

NormArgs norm_args(const morpho_layer_norm_t* p) {
    NormArgs a{};
    a.rows = p->rows;
    a.dim = p->dim;
    a.wtype = p->weight_type;
    a.eps = p->eps;
    a.sx = p->stride_x ? p->stride_x : p->dim;
    a.sres = p->stride_residual ? p->stride_residual : p->dim;
    a.sgy = p->stride_grad_y ? p->stride_grad_y : p->dim;
    a.sgh = p->stride_grad_h ? p->stride_grad_h : p->dim;
    return a;
}

// Calls f(VEC, NV, GROUP) as template constants for the width; false where the row is too long.
// Vectors of 16 bytes where every row allows them, else single elements.  A warp takes rows of up to
// 32 elements a lane, longer ones a CTA.
template <int VEC, class F>
bool with_width(int dim, F f) {
    constexpr int NV1 = VEC == 1 ? 8 : 8 / VEC;
    auto fits = [&](int nv, int group) { return static_cast<int64_t>(nv) * VEC * group >= dim; };
    if (fits(NV1, 32)) return f(std::integral_constant<int, NV1>(), std::integral_constant<int, 32>()), true;
    if (fits(2 * NV1, 32)) return f(std::integral_constant<int, 2 * NV1>(), std::integral_constant<int, 32>()), true;
    if (fits(4 * NV1, 32)) return f(std::integral_constant<int, 4 * NV1>(), std::integral_constant<int, 32>()), true;
    if (fits(NV1, kCta)) return f(std::integral_constant<int, NV1>(), std::integral_constant<int, kCta>()), true;
    if (fits(2 * NV1, kCta)) return f(std::integral_constant<int, 2 * NV1>(), std::integral_constant<int, kCta>()), true;
    if (fits(4 * NV1, kCta)) return f(std::integral_constant<int, 4 * NV1>(), std::integral_constant<int, kCta>()), true;
    return false;
}
static_assert(kMaxRegElems == 32, "with_width covers 8, 16 and 32 elements a thread");

// Calls f(NV, W) for the streaming kernels: up to 32 elements a lane, then 2, 4 and 8 warps to a row.
template <int VEC, class F>
int with_stream(int dim, F f) {
    constexpr int NV1 = 8 / VEC;
    using std::integral_constant;
    if (dim <= 256) return f(integral_constant<int, NV1>(), integral_constant<int, 1>());
    if (dim <= 512) return f(integral_constant<int, 2 * NV1>(), integral_constant<int, 1>());
    if (dim <= 1024) return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 1>());
    if (dim <= 2048) return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 2>());
    if (dim <= 4096) return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 4>());
    return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 8>());
}

constexpr int kStreamMaxDim = 8192;

int stream_warps(int dim) { return dim <= 1024 ? 1 : dim <= 2048 ? 2 : dim <= 4096 ? 4 : 8; }

// Whether the rows are worth a ring: four for every group of one CTA per SM.
bool streams(int64_t rows, int dim, bool vec, int sms) {
    return vec && dim <= kStreamMaxDim && rows >= 4LL * sms * (kStreamWarps / stream_warps(dim));
}

// Launches a streaming kernel: `per_sm` CTAs on every SM, as many stages as fit beside `fixed` bytes.
template <class K>
int launch_stream(K kern, const DeviceInfo& dev, NormArgs& a, int type, int tensors, int fixed, int per_sm, int blocks, cudaStream_t stream) {
    const int stage = a.dim * dtype_bytes(type) * tensors * (kStreamWarps / stream_warps(a.dim));
    const int room = (dev.smem_optin + 1024) / per_sm - 4096 - fixed;  // 4 KB: barriers, scratch, reserved
    a.stages = std::max(1, std::min(kMaxStages, room / stage));
    // the joining of the groups' sums (two fp32 rows) lies over the rings
    const int smem = std::max(a.stages * stage + fixed, 2 * a.dim * static_cast<int>(sizeof(float)));
    if (smem > dev.smem_optin - 2048) return set_error(MORPHO_ERR_INVALID, "layer norm: dim %d needs %d bytes of shared memory", a.dim, smem);
    MORPHO_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    MORPHO_CUDA_TRY(launch_after(kern, blocks, kStreamThreads, smem, stream, a));
    return MORPHO_OK;
}

template <class T>
int forward_t(const DeviceInfo& dev, NormArgs a, int type, bool vec, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    prof_begin(stream, "layer_norm_fwd");
    if (streams(a.rows, a.dim, vec, dev.sms)) {
        MORPHO_TRY(with_stream<V>(a.dim, [&](auto nv, auto w) {
            return launch_stream(layer_norm_fwd_stream_kernel<T, decltype(nv)::value, decltype(w)::value>, dev, a, type, a.res != nullptr ? 2 : 1, 0, 2,
                                 2 * dev.sms, stream);
        }));
        MORPHO_LAUNCH_CHECK("layer_norm_fwd");
        return MORPHO_OK;
    }
    auto launch = [&](auto vecc, auto nv, auto group) {
        constexpr int VEC = decltype(vecc)::value, NV = decltype(nv)::value, GROUP = decltype(group)::value;
        const unsigned grid = GROUP == 32 ? (a.rows + kWarpsPerCta - 1) / kWarpsPerCta : a.rows;
        layer_norm_fwd_kernel<T, VEC, NV, GROUP><<<grid, GROUP == 32 ? 32 * kWarpsPerCta : kCta, 0, stream>>>(a);
    };
    const bool done = vec ? with_width<V>(a.dim, [&](auto nv, auto g) { launch(std::integral_constant<int, V>(), nv, g); })
                          : with_width<1>(a.dim, [&](auto nv, auto g) { launch(std::integral_constant<int, 1>(), nv, g); });
    if (!done) layer_norm_fwd_long_kernel<T><<<static_cast<unsigned>(a.rows), kCta, 0, stream>>>(a);
    MORPHO_LAUNCH_CHECK("layer_norm_fwd");
    return MORPHO_OK;
}

// CTAs per SM of the streaming backward: its sums take too many registers for two above 512 columns.
int bwd_per_sm(int dim) { return dim <= 512 ? 2 : 1; }

// Partial rows (CTAs) of the backward: enough CTAs to fill the GPU, no more than there are rows.
int bwd_blocks(int64_t rows, int dim, bool stream, int sms) {
    if (stream) return bwd_per_sm(dim) * sms;
    const int64_t per = dim <= 32 * kMaxRegElems ? kWarpsPerCta : 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, 3 * sms)));
}

template <class T>
int backward_t(const DeviceInfo& dev, NormArgs a, int type, bool vec, int blocks, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    prof_begin(stream, "layer_norm_bwd");
    if (streams(a.rows, a.dim, vec, dev.sms)) {
        MORPHO_TRY(with_stream<V>(a.dim, [&](auto nv, auto w) {
            return launch_stream(layer_norm_bwd_stream_kernel<T, decltype(nv)::value, decltype(w)::value>, dev, a, type, a.gh != nullptr ? 3 : 2,
                                 a.dim * static_cast<int>(sizeof(float)), bwd_per_sm(a.dim), blocks, stream);
        }));
        MORPHO_LAUNCH_CHECK("layer_norm_bwd");
        return MORPHO_OK;
    }
    auto launch = [&](auto vecc, auto nv, auto group) {
        constexpr int VEC = decltype(vecc)::value, NV = decltype(nv)::value, GROUP = decltype(group)::value;
        const int smem = GROUP == 32 ? 2 * a.dim * static_cast<int>(sizeof(float)) : 0;
        layer_norm_bwd_kernel<T, VEC, NV, GROUP>
            <<<blocks, GROUP == 32 ? 32 * kWarpsPerCta : kCta, smem, stream>>>(a);
    };
    const bool done = vec ? with_width<V>(a.dim, [&](auto nv, auto g) { launch(std::integral_constant<int, V>(), nv, g); })
                          : with_width<1>(a.dim, [&](auto nv, auto g) { launch(std::integral_constant<int, 1>(), nv, g); });
    if (!done) {
        layer_norm_bwd_long_kernel<T><<<static_cast<unsigned>(a.rows), kCta, 0, stream>>>(a);
        if (a.part != nullptr) {
            count_launch();
            const dim3 grid((a.dim + kCta - 1) / kCta, blocks);
            layer_norm_bwd_cols_kernel<T><<<grid, kCta, 0, stream>>>(a, (a.rows + blocks - 1) / blocks);
        }
    }
    MORPHO_LAUNCH_CHECK("layer_norm_bwd");
    return MORPHO_OK;
}

int reduce_partials(const NormArgs& a, int n, void* dweight, void* dbias, cudaStream_t stream) {
    prof_begin(stream, "layer_norm_reduce");
    MORPHO_CUDA_TRY(launch_after(layer_norm_reduce_kernel, (2 * a.dim + 31) / 32, 1024, 0, stream, a.part, n, a.dim, a.wtype, dweight, dbias));
    MORPHO_LAUNCH_CHECK("layer_norm_reduce");
    return MORPHO_OK;
}

int check_norm_ptr(const void* p, const char* name, int type) {
    if (p == nullptr) return set_error(MORPHO_ERR_INVALID, "layer norm: %s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % dtype_bytes(type) != 0)
        return set_error(MORPHO_ERR_INVALID, "layer norm: %s is not aligned to its element type", name);
    return MORPHO_OK;
}

}  // namespace
}  // namespace morpho

using namespace morpho;

extern "C" MORPHO_API int morpho_sm100_layer_norm_forward(const morpho_layer_norm_t* p, const void* x,
                                                          const void* residual, const void* weight, const void* bias,
                                                          void* y, void* h, float* mean, float* rstd, void* stream) {
    clear_error();
    reset_launch_count();
    MORPHO_TRY(validate_norm(p));
    if (p->rows == 0) return MORPHO_OK;
    MORPHO_TRY(check_norm_ptr(x, "x", p->type));
    MORPHO_TRY(check_norm_ptr(y, "y", p->type));
    if (residual != nullptr) {
        MORPHO_TRY(check_norm_ptr(residual, "residual", p->type));
        MORPHO_TRY(check_norm_ptr(h, "h", p->type));
    }
    MORPHO_TRY(check_norm_ptr(mean, "mean", MORPHO_DTYPE_F32));
    MORPHO_TRY(check_norm_ptr(rstd, "rstd", MORPHO_DTYPE_F32));
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    NormArgs a = norm_args(p);
    a.status = dev.status;
    a.x = x;
    a.res = residual;
    a.w = weight;
    a.b = bias;
    a.y = y;
    a.h = h;
    a.mean = mean;
    a.rstd = rstd;
    const bool vec = p->dim * dtype_bytes(p->type) % 16 == 0 && rows_aligned(x, a.sx, p->type) &&
                     rows_aligned(residual, a.sres, p->type) && aligned16(y) && (residual == nullptr || aligned16(h));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->type == MORPHO_DTYPE_F16) return forward_t<__half>(dev, a, p->type, vec, st);
    if (p->type == MORPHO_DTYPE_BF16) return forward_t<__nv_bfloat16>(dev, a, p->type, vec, st);
    return forward_t<float>(dev, a, p->type, vec, st);
}

extern "C" MORPHO_API size_t morpho_sm100_layer_norm_backward_workspace_size(const morpho_layer_norm_t* p) {
    clear_error();
    if (validate_norm(p) != MORPHO_OK) return 0;
    DeviceInfo dev;
    const int sms = current_device_info(&dev) == MORPHO_OK ? dev.sms : 148;
    clear_error();
    return static_cast<size_t>(std::max(bwd_blocks(p->rows, p->dim, false, sms), bwd_blocks(p->rows, p->dim, true, sms))) * 2 * p->dim * sizeof(float) + 256;
}

extern "C" MORPHO_API int morpho_sm100_layer_norm_backward(const morpho_layer_norm_t* p, const void* grad_y,
                                                           const void* grad_h, const void* h, const void* weight,
                                                           const float* mean, const float* rstd, void* dx,
                                                           void* dweight, void* dbias, void* workspace,
                                                           size_t workspace_bytes, void* stream) {
    clear_error();
    reset_launch_count();
    MORPHO_TRY(validate_norm(p));
    const bool sums = dweight != nullptr || dbias != nullptr;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->rows == 0) {
        const size_t bytes = static_cast<size_t>(p->dim) * dtype_bytes(p->weight_type);
        if (dweight != nullptr) MORPHO_CUDA_TRY(cudaMemsetAsync(dweight, 0, bytes, st));
        if (dbias != nullptr) MORPHO_CUDA_TRY(cudaMemsetAsync(dbias, 0, bytes, st));
        return MORPHO_OK;
    }
    MORPHO_TRY(check_norm_ptr(grad_y, "grad_y", p->type));
    if (grad_h != nullptr) MORPHO_TRY(check_norm_ptr(grad_h, "grad_h", p->type));
    MORPHO_TRY(check_norm_ptr(h, "h", p->type));
    MORPHO_TRY(check_norm_ptr(mean, "mean", MORPHO_DTYPE_F32));
    MORPHO_TRY(check_norm_ptr(rstd, "rstd", MORPHO_DTYPE_F32));
    MORPHO_TRY(check_norm_ptr(dx, "dx", p->type));
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    NormArgs a = norm_args(p);
    const bool vec = p->dim * dtype_bytes(p->type) % 16 == 0 && rows_aligned(h, a.sx, p->type) &&
                     rows_aligned(grad_y, a.sgy, p->type) && rows_aligned(grad_h, a.sgh, p->type) && aligned16(dx);
    const int blocks = bwd_blocks(p->rows, p->dim, streams(p->rows, p->dim, vec, dev.sms), dev.sms);
    const size_t need = static_cast<size_t>(blocks) * 2 * p->dim * sizeof(float);
    if (sums) {
        MORPHO_TRY(check_norm_ptr(workspace, "workspace", MORPHO_DTYPE_F32));
        if (workspace_bytes < need)
            return set_error(MORPHO_ERR_WORKSPACE, "layer norm workspace too small: %zu < %zu bytes", workspace_bytes, need);
    }
    a.status = dev.status;
    a.x = h;
    a.w = weight;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.gy = grad_y;
    a.gh = grad_h;
    a.dx = dx;
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    int rc;
    if (p->type == MORPHO_DTYPE_F16)
        rc = backward_t<__half>(dev, a, p->type, vec, blocks, st);
    else if (p->type == MORPHO_DTYPE_BF16)
        rc = backward_t<__nv_bfloat16>(dev, a, p->type, vec, blocks, st);
    else
        rc = backward_t<float>(dev, a, p->type, vec, blocks, st);
    if (rc != MORPHO_OK || !sums) return rc;
    return reduce_partials(a, blocks, dweight, dbias, st);
}
