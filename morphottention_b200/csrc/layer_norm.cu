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
// A group of threads (8 lanes to a CTA) holds its row in registers from the load to the store.  The forward
// needs no more than that: with one row per group, many groups to an SM keep enough bytes in flight.
// The backward is persistent: each group walks rows with the stride of the grid and keeps the dweight /
// dbias sums of its columns in registers over all of them; the CTA's groups join theirs in a fixed order and
// write one fp32 partial row per CTA, which a second kernel sums in a fixed order (no atomics: the same
// bits every run).  Those sums, two fp32 registers per column, leave room for few warps, so above 256
// columns the rows in flight are bulk copies into a ring in shared memory instead (the streaming kernel).
// Rows longer than a CTA's registers hold (dim > 8192) are read again from L2.
//
// Measured, with a residual, forward and backward: 65536 x 2048 bf16 375 to 396 us on several B200s (5.4 to 5.7 TB/s, 83 to
// 88 % of a plain copy); 12608 x 768 fp16 41 us (155 MB, 3.8 TB/s: launch, filling the ring and joining the sums are
// 9 us of it).
#include <algorithm>
#include <initializer_list>

#include "elem.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace morpho {
namespace {

constexpr int kCta = 256;       // threads of the kernels for any dim, and of the widest groups
constexpr int kSmallCta = 128;  // threads of the other kernels

constexpr uint32_t K_NORM = 7;   // kernel id in the device status word

struct NormArgs {
    int64_t rows;
    int dim, wtype;
    bool wvec;  // weight and bias start on 16-byte boundaries
    float eps;
    int64_t sx, sres, sgy, sgh;  // row strides in elements
    const void *x, *res, *w, *b; // forward inputs (x is h in the backward)
    void *y, *h;
    float *mean, *rstd;
    const void *gy, *gh;
    void* dx;
    float* part;  // [grid][2][dim] partial dweight / dbias
    uint32_t* status;
    int stages;   // rows in flight per group of the streaming kernel
    int mis;      // shifted rows: elements by which the tensors' bases miss a 16-byte boundary
};

// Threads of a CTA that works in groups of GROUP threads to a row.
__host__ __device__ constexpr int cta_of(int group) { return group > kSmallCta ? group : kSmallCta; }

// Sum of two values over the group; every thread of it gets the result.  Groups of more than a warp are the
// whole CTA and use `scratch` (16 float2, used alternately by `turn`, so that one barrier per call suffices).
template <int GROUP>
__device__ __forceinline__ float2 group_sum(float a, float b, float2* scratch, int turn) {
#pragma unroll
    for (int o = (GROUP < 32 ? GROUP : 32) / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (GROUP <= 32) return make_float2(a, b);
    float2* s = scratch + (turn & 1) * 8;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 r = s[0];
#pragma unroll
    for (int i = 1; i < GROUP / 32; ++i) {
        r.x += s[i].x;
        r.y += s[i].y;
    }
    return r;
}

// VEC elements of the weight or bias from column c on (`none` where there is none).
template <int VEC>
__device__ __forceinline__ void load_param(const void* p, const NormArgs& a, int c, float none, float* out) {
    if (p == nullptr) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[k] = none;
    } else if constexpr (VEC == 1) {
        out[0] = load_as_f32(p, a.wtype, c);
    } else {
        load_n_as_f32<VEC>(p, a.wtype, c, a.wvec, out);
    }
}

// NV packs of VEC elements per thread: pack i of thread l starts at column (i * GROUP + l) * VEC.  A CTA
// has cta_of(GROUP) / GROUP rows; those past the end read the last row again and write nothing.
template <class T, int VEC, int NV, int GROUP>
__global__ void __launch_bounds__(cta_of(GROUP)) layer_norm_fwd_kernel(const NormArgs a) {
    __shared__ float2 scratch[16];
    pdl_release();
    pdl_wait();
    constexpr int ROWS = cta_of(GROUP) / GROUP;
    const int l = threadIdx.x % GROUP;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / GROUP;
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
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
            if (live) store_pack<T, VEC>(h + c, px[i]);
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
    if (!live) return;
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
        float w[VEC], b[VEC];
        load_param<VEC>(a.w, a, c, 1.f, w);
        load_param<VEC>(a.b, a, c, 0.f, b);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = from_f32<T>(fmaf(v[i * VEC + k] * r, w[k], b[k]));
        store_pack<T, VEC>(y + c, o);
    }
}

// ---- shifted rows: contiguous rows whose length is no multiple of 16 bytes ---------------------------------
// All tensors are contiguous and miss a 16-byte boundary by the same number of elements, so a row begins
// `off` elements into an aligned pack, in every tensor the same: packs are moved whole, the elements of the
// first and the last that belong to the neighbours are masked, and only weight and bias are indexed by the
// true column (from shared memory, one float in nine left out so that the lanes' strides hit all banks).

template <int VEC>
__device__ __forceinline__ int row_offset(const NormArgs& a, int64_t row) {
    return (a.mis + static_cast<int>(row % VEC) * (a.dim % VEC)) % VEC;
}

__host__ __device__ constexpr int param_at(int c) { return c + 8 + ((c + 8) >> 3); }  // c >= -8

template <int VEC, class T>
__device__ __forceinline__ void store_cols(T* at, const Pack<T, VEC>& p, int col, int dim) {
    if (col >= 0 && col + VEC <= dim) {
        store_pack<T, VEC>(at, p);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (col + k >= 0 && col + k < dim) at[k] = p.v[k];
    }
}

template <class T, int NV, int GROUP>
__global__ void __launch_bounds__(cta_of(GROUP)) layer_norm_fwd_shift_kernel(const NormArgs a) {
    constexpr int VEC = 16 / sizeof(T), ROWS = cta_of(GROUP) / GROUP;
    extern __shared__ float ws[];  // weight, then bias
    __shared__ float2 scratch[16];
    pdl_release();
    pdl_wait();
    const int l = threadIdx.x % GROUP, g = threadIdx.x / GROUP;
    const int width = param_at(a.dim + 8);
    for (int c = static_cast<int>(threadIdx.x) - 8; c < a.dim + 8; c += cta_of(GROUP)) {
        const bool in = c >= 0 && c < a.dim;
        ws[param_at(c)] = a.w != nullptr && in ? load_as_f32(a.w, a.wtype, c) : 1.f;
        ws[width + param_at(c)] = a.b != nullptr && in ? load_as_f32(a.b, a.wtype, c) : 0.f;
    }
    __syncthreads();
    const float inv = 1.0f / static_cast<float>(a.dim);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS; base < a.rows; base += static_cast<int64_t>(gridDim.x) * ROWS) {
        const bool live = base + g < a.rows;
        const int64_t row = live ? base + g : a.rows - 1;
        const int off = row_offset<VEC>(a, row);
        const int64_t at = row * a.dim - off;  // an aligned pack
        Pack<T, VEC> px[NV], pr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * GROUP + l) * VEC;
            if (j - off < a.dim) {
                px[i] = load_pack<T, VEC>(static_cast<const T*>(a.x) + at + j);
                if (a.res != nullptr) pr[i] = load_pack<T, VEC>(static_cast<const T*>(a.res) + at + j);
            }
        }
        float v[NV * VEC];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * GROUP + l) * VEC, col = j - off;
            if (a.res != nullptr && col < a.dim) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) px[i].v[k] = from_f32<T>(to_f32(px[i].v[k]) + to_f32(pr[i].v[k]));
                if (live) store_cols<VEC>(static_cast<T*>(a.h) + at + j, px[i], col, a.dim);
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[i * VEC + k] = col + k >= 0 && col + k < a.dim ? to_f32(px[i].v[k]) : 0.f;
                sum += v[i * VEC + k];
            }
        }
        const float mu = group_sum<GROUP>(sum, 0.f, scratch, 0).x * inv;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * GROUP + l) * VEC - off;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[i * VEC + k] -= mu;
                if (col + k >= 0 && col + k < a.dim) sq = fmaf(v[i * VEC + k], v[i * VEC + k], sq);
            }
        }
        const float r = rsqrtf(group_sum<GROUP>(sq, 0.f, scratch, 1).x * inv + a.eps);
        if (live && l == 0) {
            a.mean[row] = mu;
            a.rstd[row] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * GROUP + l) * VEC, col = j - off;
            if (col < a.dim && live) {
                Pack<T, VEC> o;
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    o.v[k] = from_f32<T>(fmaf(v[i * VEC + k] * r, ws[param_at(col + k)], ws[width + param_at(col + k)]));
                store_cols<VEC>(static_cast<T*>(a.y) + at + j, o, col, a.dim);
            }
        }
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

// The dweight / dbias sums of a CTA's GROUPS groups of G threads, each with NV packs of VEC columns a
// thread, joined in the groups' order and written to `part` [2][dim].  Shared memory: sums_floats() floats.
// Element (i, k) of thread l stands at (i VEC + k) (G + 1) + l, so that neither side conflicts on a bank.
__host__ __device__ constexpr int sums_floats(int elems, int group, int groups) { return 2 * groups * elems * (group + 1); }

// Column c of group i is element c + off(i) of its packs.
template <int VEC, int NV, int G, int GROUPS, class Off>
__device__ __forceinline__ void join_sums(float* sums, const float* dw, const float* db, int dim, float* part, Off off) {
    constexpr int E = NV * VEC, SIZE = E * (G + 1);
    const int l = threadIdx.x % G, g = threadIdx.x / G;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        sums[(2 * g) * SIZE + e * (G + 1) + l] = dw[e];
        sums[(2 * g + 1) * SIZE + e * (G + 1) + l] = db[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * dim; c += G * GROUPS) {
        const int which = c >= dim, col = which ? c - dim : c;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int e = col + off(i), k = e % VEC, t = e / VEC;
            s += sums[(2 * i + which) * SIZE + ((t / G) * VEC + k) * (G + 1) + t % G];
        }
        part[c] = s;
    }
}

template <class T, int VEC, int NV, int GROUP>
__global__ void __launch_bounds__(cta_of(GROUP), NV * VEC <= 8 && GROUP <= 32 ? 5 : 1) layer_norm_bwd_kernel(const NormArgs a) {
    constexpr int E = NV * VEC, ROWS = cta_of(GROUP) / GROUP;
    __shared__ float2 scratch[16];
    extern __shared__ float sums[];
    pdl_release();
    pdl_wait();
    const int l = threadIdx.x % GROUP, g = threadIdx.x / GROUP;
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
    float dw[E], db[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    const float inv = 1.0f / static_cast<float>(a.dim);
    int turn = 0;
    // the CTA's rows go together; those past the end read the last row again and add nothing
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS; base < a.rows; base += step, ++turn) {
        const bool live = base + g < a.rows;
        const int64_t row = live ? base + g : a.rows - 1;
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
        float xh[E], gw[E];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * GROUP + l) * VEC;
            if (c < a.dim) {
                float w[VEC];
                load_param<VEC>(a.w, a, c, 1.f, w);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    const float d = live ? to_f32(pg[i].v[k]) : 0.f;
                    xh[e] = (to_f32(ph[i].v[k]) - mu) * r;
                    if (live) dw[e] = fmaf(d, xh[e], dw[e]);
                    db[e] += d;
                    gw[e] = d * w[k];
                    s0 += gw[e];
                    s1 = fmaf(gw[e], xh[e], s1);
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
            if (c >= a.dim || !live) continue;
            Pack<T, VEC> o, pd;
            if (gh != nullptr) pd = load_pack<T, VEC>(gh + c);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const int e = i * VEC + k;
                float d = r * (gw[e] - mg - xh[e] * mgx);
                if (gh != nullptr) d += to_f32(pd.v[k]);
                o.v[k] = from_f32<T>(d);
            }
            store_pack<T, VEC>(dx + c, o);
        }
    }
    if (a.part == nullptr) return;
    join_sums<VEC, NV, GROUP, ROWS>(sums, dw, db, a.dim, a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.dim, [](int) { return 0; });
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

// ---- the streaming backward: up to 32 elements a lane --------------------------------------------------

constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = 32 * kStreamWarps;
constexpr int kMaxStages = 8;

// Sums of two values over the W warps of a group (threads 32 W of the CTA, group `g`).  `ok`, which is uniform in
// each warp, comes back as whether it holds in all of them: the group goes on or gives up as one.
template <int W>
__device__ __forceinline__ float2 warps_sum(float a, float b, bool& ok, float2 (*scratch)[kStreamWarps], int turn, int g) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (W == 1) return make_float2(a, b);
    float2* s = scratch[turn & 1] + g * W;
    if ((threadIdx.x & 31) == 0) s[(threadIdx.x >> 5) & (W - 1)] = make_float2(a, b);
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(all)
        : "r"(static_cast<uint32_t>(ok)), "r"(1 + g), "n"(32 * W)
        : "memory");
    ok = all != 0u;
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

    // One thread: fetch `bytes` of one row of the given tensors (c NULL: two) as use number i of the ring.
    __device__ void fetch(int i, const void* a, const void* b, const void* c, uint32_t bytes) const {
        const int s = i % stages;
        const uint32_t bar = bars + 8 * s, dst = data + s * stage_bytes;
        mbar_arrive_expect_tx(bar, bytes * (2 + (c != nullptr)));
        bulk_load(dst, a, bytes, bar);
        bulk_load(dst + row_bytes, b, bytes, bar);
        if (c != nullptr) bulk_load(dst + 2 * row_bytes, c, bytes, bar);
    }
    // One thread, after the group gave up at use i: the n copies from there on that may still be in flight, each
    // waited for in turn.
    __device__ void drain(int i, int n, uint32_t* status) const {
        for (int k = i; k < i + n; ++k) mbar_wait(bars + 8 * (k % stages), (k / stages) & 1, status, K_NORM, 3);
    }
    __device__ uint32_t stage(int i) const { return data + (i % stages) * stage_bytes; }
    // A whole warp.
    __device__ bool wait(int i, uint32_t* status) const {
        return mbar_wait_warp(bars + 8 * (i % stages), (i / stages) & 1, status, K_NORM, 2);
    }
};

template <class T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> shared_pack(uint32_t addr) {
    const uint4 x = ld_shared_u4(addr);
    return *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(&x);
}

// Bytes of a row in the ring: shifted rows are fetched from the boundary before to the one after.
__host__ __device__ constexpr int stream_row_bytes(int dim, int size, bool shift) {
    return shift ? (dim + 2 * (16 / size) - 2) / (16 / size) * 16 : dim * size;
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

// SHIFT: shifted rows (above); the number of groups is then a multiple of VEC or covers the rows, so that
// all rows of a group begin at one offset and its sums belong to the same columns throughout.
template <class T, int NV, int W, bool SHIFT>
__global__ void __launch_bounds__(kStreamThreads, NV * 16 / sizeof(T) > 16 ? 1 : 2) layer_norm_bwd_stream_kernel(const NormArgs a) {
    constexpr int VEC = 16 / sizeof(T), E = NV * VEC, G = 32 * W, GROUPS = kStreamWarps / W;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[GROUPS * kMaxStages];
    __shared__ float2 scratch[2][kStreamWarps];
    pdl_release();
    const int l = threadIdx.x % G, g = threadIdx.x / G;
    const int tensors = a.gh != nullptr ? 3 : 2;
    const RowRing ring = make_ring<W>(smem, bars, a, stream_row_bytes(a.dim, sizeof(T), SHIFT), tensors);
    float* ws = reinterpret_cast<float*>(smem + GROUPS * a.stages * ring.stage_bytes);  // the weight, fp32
    pdl_wait();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * GROUPS + g, step = static_cast<int64_t>(gridDim.x) * GROUPS;
    const T *h = static_cast<const T*>(a.x), *gy = static_cast<const T*>(a.gy), *gh = static_cast<const T*>(a.gh);
    const int off = SHIFT ? row_offset<VEC>(a, first) : 0;
    const uint32_t bytes = SHIFT ? static_cast<uint32_t>((a.dim + off + VEC - 1) / VEC * 16) : ring.row_bytes;
    auto fetch = [&](int i, int64_t row) {
        if (row < a.rows)
            ring.fetch(i, h + row * a.sx - off, gy + row * a.sgy - off, gh != nullptr ? gh + row * a.sgh - off : nullptr, bytes);
    };
    if (l == 0)
        for (int i = 0; i < a.stages; ++i) fetch(i, first + i * step);
    if (SHIFT) {
        for (int c = static_cast<int>(threadIdx.x) - 8; c < a.dim + 8; c += kStreamThreads)
            ws[param_at(c)] = a.w != nullptr && c >= 0 && c < a.dim ? load_as_f32(a.w, a.wtype, c) : 1.f;
    } else {
        for (int c = threadIdx.x * VEC; c < a.dim; c += kStreamThreads * VEC) {
            float w[VEC];
            load_param<VEC>(a.w, a, c, 1.f, w);
#pragma unroll
            for (int k = 0; k < VEC; ++k) ws[c + k] = w[k];
        }
    }
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
        bool ok = ring.wait(i, a.status);  // (if not, what follows up to the sums works on what lies there)
        const uint32_t src = ring.stage(i);
        float s0 = 0.f, s1 = 0.f;
        float xh[E], gw[E];
        Pack<T, VEC> ph[NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + l) * VEC, col = c - off;
            if (col < a.dim) {
                const Pack<T, VEC> p = shared_pack<T>(src + c * sizeof(T)), q = shared_pack<T>(src + ring.row_bytes + c * sizeof(T));
                if (gh != nullptr) ph[n] = shared_pack<T>(src + 2 * ring.row_bytes + c * sizeof(T));
                float w[VEC];
                if (SHIFT) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) w[k] = ws[param_at(col + k)];
                } else {
#pragma unroll
                    for (int k = 0; k < VEC; k += 4) {
                        const float4 w4 = *reinterpret_cast<const float4*>(ws + c + k);
                        w[k] = w4.x, w[k + 1] = w4.y, w[k + 2] = w4.z, w[k + 3] = w4.w;
                    }
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = n * VEC + k;
                    const bool in = !SHIFT || (col + k >= 0 && col + k < a.dim);
                    const float d = in ? to_f32(q.v[k]) : 0.f;
                    xh[e] = in ? (to_f32(p.v[k]) - mu) * r : 0.f;
                    dw[e] = fmaf(d, xh[e], dw[e]);
                    db[e] += d;
                    gw[e] = d * w[k];
                    s0 += gw[e];
                    s1 = fmaf(gw[e], xh[e], s1);
                }
            }
        }
        const float2 s = warps_sum<W>(s0, s1, ok, scratch, i, g);
        if (!ok) {
            int fetched = 0;
            while (fetched < a.stages && row + fetched * step < a.rows) ++fetched;
            if (l == 0) ring.drain(i, fetched, a.status);
            break;
        }
        __syncwarp();
        if (l == 0) fetch(i + a.stages, row + a.stages * step);
        const float mg = s.x * inv, mgx = s.y * inv;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + l) * VEC, col = c - off;
            if (col < a.dim) {
                Pack<T, VEC> o;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = n * VEC + k;
                    float d = r * (gw[e] - mg - xh[e] * mgx);
                    if (gh != nullptr) d += to_f32(ph[n].v[k]);
                    o.v[k] = from_f32<T>(d);
                }
                T* at = static_cast<T*>(a.dx) + row * a.dim + col;
                if (SHIFT)
                    store_cols<VEC>(at, o, col, a.dim);
                else
                    store_pack<T, VEC>(at, o);
            }
        }
        mu = mu1;
        r = r1;
    }
    if (a.part == nullptr) return;
    __syncthreads();  // over the rings: every fetched row has been waited for
    join_sums<VEC, NV, G, GROUPS>(reinterpret_cast<float*>(smem), dw, db, a.dim, a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.dim,
                                  [&](int i) { return SHIFT ? row_offset<VEC>(a, static_cast<int64_t>(blockIdx.x) * GROUPS + i) : 0; });
}

// Self-test of giving up: the second warp of group 1 waits for a row that is never fetched, the first did not have
// to; seen[w]: what warp w was told (all groups but that one go on).
__global__ void __launch_bounds__(kStreamThreads) row_wait_kernel(const NormArgs a, uint32_t* seen) {
    constexpr int W = 2;
    __shared__ __align__(128) uint8_t smem[16 * 2 * kStreamWarps / W];
    __shared__ uint64_t bars[kStreamWarps / W * kMaxStages];
    __shared__ float2 scratch[2][kStreamWarps];
    const RowRing ring = make_ring<W>(smem, bars, a, 16, 2);
    const int g = threadIdx.x / (32 * W), warp = threadIdx.x >> 5;
    bool ok = g != 1 || warp % W == 0 || ring.wait(0, a.status);
    const float2 s = warps_sum<W>(1.f, 2.f, ok, scratch, 0, g);
    if ((threadIdx.x & 31) == 0) seen[warp] = ok && s.x == 32.f * W && s.y == 64.f * W;
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

// Calls f(NV, GROUP) as template constants for the width: groups of 8 or 16 lanes for rows that they hold
// in 8 elements a lane, a warp for up to 32 elements a lane, then 128 and 256 threads of 16 or 32 in the
// forward (65536 x 2048 bf16: 128 threads 6 TB/s, a warp with 64 elements a lane 5; the backward streams there).  Rows of single elements (VEC 1, unaligned) go to 256
// threads above 256 columns: their many loads are better spread.  False where the row is too long.
template <int VEC, bool FORWARD, class F>
bool with_width(int dim, F f) {
    using std::integral_constant;
    constexpr int N = VEC == 1 ? 8 : 8 / VEC;  // packs of 8 elements
#define MORPHO_TRY_WIDTH(packs, group) \
    if (static_cast<int64_t>(packs) * VEC * (group) >= dim) return f(integral_constant<int, packs>(), integral_constant<int, group>()), true
    MORPHO_TRY_WIDTH(N, 8);
    MORPHO_TRY_WIDTH(N, 16);
    MORPHO_TRY_WIDTH(N, 32);
    if constexpr (VEC == 1) {
        MORPHO_TRY_WIDTH(N, kCta);
        MORPHO_TRY_WIDTH(2 * N, kCta);
    } else {
        MORPHO_TRY_WIDTH(2 * N, 32);
        MORPHO_TRY_WIDTH(4 * N, 32);
    }
    if constexpr (FORWARD && VEC > 1) {
        MORPHO_TRY_WIDTH(2 * N, kSmallCta);
        MORPHO_TRY_WIDTH(4 * N, kSmallCta);
    }
    if constexpr (FORWARD || VEC == 1) MORPHO_TRY_WIDTH(4 * N, kCta);
#undef MORPHO_TRY_WIDTH
    return false;
}

// Calls f(NV, W) for the streaming backward: up to 32 elements a lane, then 2, 4 and 8 warps to a row.
template <int VEC, bool SHIFT, class F>
int with_stream(int dim, F f) {
    constexpr int NV1 = 8 / VEC;
    using std::integral_constant;
    if constexpr (SHIFT) {
        dim += VEC - 1;
        if (dim <= 256) return f(integral_constant<int, NV1>(), integral_constant<int, 1>());
    }
    if (dim <= 512) return f(integral_constant<int, 2 * NV1>(), integral_constant<int, 1>());
    if (dim <= 1024) return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 1>());
    if (dim <= 2048) return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 2>());
    if (dim <= 4096) return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 4>());
    return f(integral_constant<int, 4 * NV1>(), integral_constant<int, 8>());
}

// How a call's rows lie: on 16-byte boundaries, shifted (contiguous, all tensors alike), or anyhow.
enum class Rows { kAligned, kShifted, kAny };

constexpr int kMaxDim = 8192;                      // columns that registers hold
constexpr int kShiftMaxDim = kMaxDim - 7;          // and with the widest offset
constexpr int kStreamMinDim = 264;

int stream_warps(int width) { return width <= 1024 ? 1 : width <= 2048 ? 2 : width <= 4096 ? 4 : 8; }

// CTAs per SM of the streaming backward: its sums take too many registers for two above 512 columns.
int stream_per_sm(int width) { return width <= 512 ? 2 : 1; }

// Columns and the widest offset.
int stream_width(int dim, Rows how, int type) { return dim + (how == Rows::kShifted ? 16 / dtype_bytes(type) - 1 : 0); }

// Whether the backward streams: aligned rows up to 256 columns do not (a lane's eight sums leave room for so
// many warps that plain loads do as well: 12608 x 256 fp16 11.7 us, not 11.5); above 1024 it always pays, in
// between from one row for every group on (1184 x 1024: 7.4 us, not 8.5; with half the groups idle it loses).
bool streams(int64_t rows, int dim, Rows how, int sms) {
    if (how == Rows::kAny || dim > (how == Rows::kShifted ? kShiftMaxDim : kMaxDim)) return false;
    if (how == Rows::kAligned && dim < kStreamMinDim) return false;
    return dim > 1024 || rows >= static_cast<int64_t>(sms) * kStreamWarps;
}

// Launches a streaming kernel: `per_sm` CTAs on every SM, as many stages as fit beside `fixed` bytes, `join`
// bytes at the end.
template <class K>
int launch_stream(K kern, SharedLimit& limit, const DeviceInfo& dev, NormArgs& a, int row_bytes, int tensors, int groups, int fixed, int join, int per_sm, int blocks,
                  cudaStream_t stream) {
    const int stage = row_bytes * tensors * groups;
    const int room = (dev.smem_optin + 1024) / per_sm - 4096 - fixed;  // 4 KB: barriers, scratch, reserved
    a.stages = std::max(1, std::min(kMaxStages, room / stage));
    const int smem = std::max(a.stages * stage + fixed, join);  // the joining of the groups' sums lies over the rings
    if (smem > dev.smem_optin - 2048) return set_error(MORPHO_ERR_INVALID, "layer norm: dim %d needs %d bytes of shared memory", a.dim, smem);
    MORPHO_CUDA_TRY(limit.raise(kern, dev.device, smem));
    MORPHO_CUDA_TRY(launch_after(kern, blocks, kStreamThreads, smem, stream, a));
    return MORPHO_OK;
}

template <class T>
int forward_t(const DeviceInfo& dev, const NormArgs& a, Rows how, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    prof_begin(stream, "layer_norm_fwd");
    cudaError_t e = cudaSuccess;
    auto go = [&](auto vecc) {
        constexpr int VEC = decltype(vecc)::value;
        return with_width<VEC, true>(a.dim, [&](auto nv, auto group) {
            constexpr int NV = decltype(nv)::value, GROUP = decltype(group)::value;
            const int64_t rows = cta_of(GROUP) / GROUP;
            e = launch_after(layer_norm_fwd_kernel<T, VEC, NV, GROUP>, static_cast<unsigned>((a.rows + rows - 1) / rows), cta_of(GROUP), 0, stream, a);
        });
    };
    bool done;
    // (a shifted kernel lays weight and bias out in shared memory first: for many rows)
    if (how == Rows::kShifted && a.dim <= kShiftMaxDim && a.rows >= static_cast<int64_t>(dev.sms) * 8) {
        done = with_width<V, true>(a.dim + V - 1, [&](auto nv, auto group) {
            constexpr int NV = decltype(nv)::value, GROUP = decltype(group)::value;
            const int64_t rows = cta_of(GROUP) / GROUP;
            const int smem = 2 * param_at(a.dim + 8) * static_cast<int>(sizeof(float));
            const int64_t most = static_cast<int64_t>(dev.sms) * std::max(1, std::min(4 * kSmallCta / cta_of(GROUP), 200 * 1024 / (smem + 1024)));
            auto kern = layer_norm_fwd_shift_kernel<T, NV, GROUP>;
            static SharedLimit limit;
            e = limit.raise(kern, dev.device, smem);
            if (e == cudaSuccess) e = launch_after(kern, static_cast<unsigned>(std::min((a.rows + rows - 1) / rows, most)), cta_of(GROUP), smem, stream, a);
        });
    } else {
        done = how == Rows::kAligned ? go(std::integral_constant<int, V>()) : go(std::integral_constant<int, 1>());
    }
    if (!done) layer_norm_fwd_long_kernel<T><<<static_cast<unsigned>(a.rows), kCta, 0, stream>>>(a);
    MORPHO_CUDA_TRY(e);
    MORPHO_LAUNCH_CHECK("layer_norm_fwd");
    return MORPHO_OK;
}

// Partial rows (CTAs) of the backward: enough CTAs to fill the GPU, no more than the rows need.
int bwd_blocks(int64_t rows, int dim, Rows how, int type, int sms) {
    int64_t per, most;  // rows at a time of a CTA; CTAs
    if (streams(rows, dim, how, sms)) {
        const int width = stream_width(dim, how, type);
        per = kStreamWarps / stream_warps(width);
        most = stream_per_sm(width) * sms;
        if (how == Rows::kShifted) most = std::max<int64_t>(8, most / 8 * 8);  // groups in multiples of a pack
    } else if (dim <= 256) {
        per = kSmallCta / (dim <= 64 ? 8 : dim <= 128 ? 16 : 32);
        most = 5 * sms;
    } else {
        per = how == Rows::kAligned && dim <= 1024 ? kSmallCta / 32 : 1;
        most = 2 * sms;
    }
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, most)));
}

template <class T, bool SHIFT>
int backward_stream(const DeviceInfo& dev, NormArgs a, int type, int blocks, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const int width = stream_width(a.dim, SHIFT ? Rows::kShifted : Rows::kAligned, type);
    return with_stream<V, SHIFT>(a.dim, [&](auto nv, auto w) {
        constexpr int NV = decltype(nv)::value, W = decltype(w)::value;
        const int join = a.part == nullptr ? 0 : static_cast<int>(sizeof(float)) * sums_floats(NV * V, 32 * W, kStreamWarps / W);
        const int fixed = static_cast<int>(sizeof(float)) * (SHIFT ? param_at(a.dim + 8) : a.dim);
        static SharedLimit limit;
        return launch_stream(layer_norm_bwd_stream_kernel<T, NV, W, SHIFT>, limit, dev, a, stream_row_bytes(a.dim, sizeof(T), SHIFT), a.gh != nullptr ? 3 : 2,
                             kStreamWarps / W, fixed, join, stream_per_sm(width), blocks, stream);
    });
}

template <class T>
int backward_t(const DeviceInfo& dev, NormArgs a, int type, Rows how, int blocks, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    prof_begin(stream, "layer_norm_bwd");
    if (streams(a.rows, a.dim, how, dev.sms)) {
        MORPHO_TRY(how == Rows::kShifted ? (backward_stream<T, true>(dev, a, type, blocks, stream)) : (backward_stream<T, false>(dev, a, type, blocks, stream)));
        MORPHO_LAUNCH_CHECK("layer_norm_bwd");
        return MORPHO_OK;
    }
    cudaError_t e = cudaSuccess;
    auto go = [&](auto vecc) {
        constexpr int VEC = decltype(vecc)::value;
        return with_width<VEC, false>(a.dim, [&](auto nv, auto group) {
            constexpr int NV = decltype(nv)::value, GROUP = decltype(group)::value;
            constexpr int smem = sums_floats(NV * VEC, GROUP, cta_of(GROUP) / GROUP) * static_cast<int>(sizeof(float));
            auto kern = layer_norm_bwd_kernel<T, VEC, NV, GROUP>;
            static SharedLimit limit;
            e = limit.raise(kern, dev.device, smem);
            if (e == cudaSuccess) e = launch_after(kern, static_cast<unsigned>(blocks), cta_of(GROUP), smem, stream, a);
        });
    };
    if (!(how == Rows::kAligned ? go(std::integral_constant<int, V>()) : go(std::integral_constant<int, 1>()))) {
        layer_norm_bwd_long_kernel<T><<<static_cast<unsigned>(a.rows), kCta, 0, stream>>>(a);
        if (a.part != nullptr) {
            count_launch();
            const dim3 grid((a.dim + kCta - 1) / kCta, blocks);
            layer_norm_bwd_cols_kernel<T><<<grid, kCta, 0, stream>>>(a, (a.rows + blocks - 1) / blocks);
        }
    }
    MORPHO_CUDA_TRY(e);
    MORPHO_LAUNCH_CHECK("layer_norm_bwd");
    return MORPHO_OK;
}

// How the rows of some tensors lie (base, row stride in elements; NULL: none); *mis for shifted ones.
struct RowsOf {
    const void* p;
    int64_t stride;
};
Rows rows_of(std::initializer_list<RowsOf> tensors, int dim, int type, int* mis) {
    const int size = dtype_bytes(type);
    bool aligned = dim * size % 16 == 0, alike = true;
    *mis = -1;
    for (const RowsOf& t : tensors) {
        if (t.p == nullptr) continue;
        aligned = aligned && rows_aligned(t.p, t.stride, type);
        const int m = static_cast<int>((reinterpret_cast<uintptr_t>(t.p) & 15u) / size);
        alike = alike && t.stride == dim && (*mis < 0 || *mis == m);
        *mis = m;
    }
    return aligned ? Rows::kAligned : alike ? Rows::kShifted : Rows::kAny;
}

int reduce_partials(const NormArgs& a, int n, void* dweight, void* dbias, cudaStream_t stream) {
    prof_begin(stream, "layer_norm_reduce");
    MORPHO_CUDA_TRY(launch_after(layer_norm_reduce_kernel, (2 * a.dim + 31) / 32, 1024, 0, stream, a.part, n, a.dim, a.wtype, dweight, dbias));
    MORPHO_LAUNCH_CHECK("layer_norm_reduce");
    return MORPHO_OK;
}

int check_norm_align(const void* p, const char* name, int type) {
    if (reinterpret_cast<uintptr_t>(p) % dtype_bytes(type) != 0)
        return set_error(MORPHO_ERR_INVALID, "layer norm: %s is not aligned to its element type", name);
    return MORPHO_OK;
}

int check_norm_ptr(const void* p, const char* name, int type) {
    if (p == nullptr) return set_error(MORPHO_ERR_INVALID, "layer norm: %s is NULL", name);
    return check_norm_align(p, name, type);
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
        const bool gaps = (h == x && p->stride_x != 0 && p->stride_x != p->dim) || (h == residual && p->stride_residual != 0 && p->stride_residual != p->dim);
        if (gaps && p->rows > 1) return set_error(MORPHO_ERR_INVALID, "layer norm: h in place needs rows without gaps");
    }
    MORPHO_TRY(check_norm_align(weight, "weight", p->weight_type));
    MORPHO_TRY(check_norm_align(bias, "bias", p->weight_type));
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
    a.wvec = aligned16(weight) && aligned16(bias);
    a.y = y;
    a.h = h;
    a.mean = mean;
    a.rstd = rstd;
    const Rows how = rows_of({{x, a.sx}, {residual, a.sres}, {y, a.dim}, {residual != nullptr ? h : nullptr, a.dim}}, p->dim, p->type, &a.mis);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->type == MORPHO_DTYPE_F16) return forward_t<__half>(dev, a, how, st);
    if (p->type == MORPHO_DTYPE_BF16) return forward_t<__nv_bfloat16>(dev, a, how, st);
    return forward_t<float>(dev, a, how, st);
}

extern "C" MORPHO_API size_t morpho_sm100_layer_norm_backward_workspace_size(const morpho_layer_norm_t* p) {
    clear_error();
    if (validate_norm(p) != MORPHO_OK) return 0;
    DeviceInfo dev;
    const int sms = current_device_info(&dev) == MORPHO_OK ? dev.sms : 148;
    clear_error();
    int blocks = 0;
    for (const Rows how : {Rows::kAligned, Rows::kShifted, Rows::kAny}) blocks = std::max(blocks, bwd_blocks(p->rows, p->dim, how, p->type, sms));
    return static_cast<size_t>(blocks) * 2 * p->dim * sizeof(float) + 256;
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
    MORPHO_TRY(check_norm_align(dweight, "dweight", p->weight_type));
    MORPHO_TRY(check_norm_align(dbias, "dbias", p->weight_type));
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
    MORPHO_TRY(check_norm_align(weight, "weight", p->weight_type));
    MORPHO_TRY(check_norm_ptr(mean, "mean", MORPHO_DTYPE_F32));
    MORPHO_TRY(check_norm_ptr(rstd, "rstd", MORPHO_DTYPE_F32));
    MORPHO_TRY(check_norm_ptr(dx, "dx", p->type));
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    NormArgs a = norm_args(p);
    const Rows how = rows_of({{h, a.sx}, {grad_y, a.sgy}, {grad_h, a.sgh}, {dx, a.dim}}, p->dim, p->type, &a.mis);
    const int blocks = bwd_blocks(p->rows, p->dim, how, p->type, dev.sms);
    const size_t need = static_cast<size_t>(blocks) * 2 * p->dim * sizeof(float);
    if (sums) {
        MORPHO_TRY(check_norm_ptr(workspace, "workspace", MORPHO_DTYPE_F32));
        if (workspace_bytes < need)
            return set_error(MORPHO_ERR_WORKSPACE, "layer norm workspace too small: %zu < %zu bytes", workspace_bytes, need);
    }
    a.status = dev.status;
    a.x = h;
    a.w = weight;
    a.wvec = aligned16(weight);
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.gy = grad_y;
    a.gh = grad_h;
    a.dx = dx;
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    int rc;
    if (p->type == MORPHO_DTYPE_F16)
        rc = backward_t<__half>(dev, a, p->type, how, blocks, st);
    else if (p->type == MORPHO_DTYPE_BF16)
        rc = backward_t<__nv_bfloat16>(dev, a, p->type, how, blocks, st);
    else
        rc = backward_t<float>(dev, a, p->type, how, blocks, st);
    if (rc != MORPHO_OK || !sums) return rc;
    return reduce_partials(a, blocks, dweight, dbias, st);
}

extern "C" MORPHO_API int morpho_sm100_selftest_row_wait(uint32_t* seen, void* stream) {
    clear_error();
    MORPHO_TRY(check_norm_ptr(seen, "seen", MORPHO_DTYPE_F32));
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    NormArgs a{};
    a.stages = 1;
    a.status = dev.status;
    row_wait_kernel<<<1, kStreamThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, seen);
    MORPHO_CUDA_TRY(cudaGetLastError());
    return MORPHO_OK;
}
