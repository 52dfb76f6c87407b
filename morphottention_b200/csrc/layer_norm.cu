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
// once.  A group of threads (a warp, or a CTA of 256 threads for long rows) holds its row in registers
// from the load to the store; the variance is the second moment about the mean it has just formed,
// which loses nothing to cancellation.  All sums are fp32.
//
// The backward is persistent: each group walks rows with the stride of the grid, keeping the dweight /
// dbias sums of its columns in registers; the CTA's groups join theirs in a fixed order and write one
// fp32 partial row per CTA, which a second kernel sums in a fixed order (no atomics: the same bits every
// run).  Rows longer than a CTA's registers hold (dim > 8192) are read again from L2 instead.
#include <algorithm>

#include "elem.cuh"
#include "kernels.h"

namespace morpho {
namespace {

constexpr int kCta = 256;        // threads per row of the CTA-wide kernels
constexpr int kWarpsPerCta = 4;  // rows at a time of the warp-wide kernels
constexpr int kMaxRegElems = 32; // row elements a thread holds

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

// dweight / dbias = the sums of the `n` partial rows, in a fixed order: 32 columns per block, eight
// threads a column.
__global__ void __launch_bounds__(kCta) layer_norm_reduce_kernel(const float* part, int n, int dim, int wtype, void* dw,
                                                                 void* db) {
    __shared__ float s[8][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + cx;
    float sum = 0.f;
    if (c < 2 * static_cast<int64_t>(dim)) {
#pragma unroll 4
        for (int i = ry; i < n; i += 8) sum += part[static_cast<int64_t>(i) * 2 * dim + c];
    }
    s[ry][cx] = sum;
    __syncthreads();
    if (ry != 0 || c >= 2 * static_cast<int64_t>(dim)) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += s[i][cx];
    if (c < dim) {
        if (dw != nullptr) store_from_f32(dw, wtype, c, sum);
    } else if (db != nullptr) {
        store_from_f32(db, wtype, c - dim, sum);
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

template <class T>
int forward_t(const NormArgs& a, bool vec, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    prof_begin(stream, "layer_norm_fwd");
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

// Partial rows (CTAs) of the backward: enough CTAs to fill the GPU, no more than there are rows.
int bwd_blocks(int64_t rows, int dim, int sms) {
    const int64_t per = dim <= 32 * kMaxRegElems ? kWarpsPerCta : 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, 3 * sms)));
}

template <class T>
int backward_t(NormArgs a, bool vec, int blocks, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    prof_begin(stream, "layer_norm_bwd");
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
    layer_norm_reduce_kernel<<<(2 * a.dim + 31) / 32, kCta, 0, stream>>>(a.part, n, a.dim, a.wtype, dweight, dbias);
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
    if (p->type == MORPHO_DTYPE_F16) return forward_t<__half>(a, vec, st);
    if (p->type == MORPHO_DTYPE_BF16) return forward_t<__nv_bfloat16>(a, vec, st);
    return forward_t<float>(a, vec, st);
}

extern "C" MORPHO_API size_t morpho_sm100_layer_norm_backward_workspace_size(const morpho_layer_norm_t* p) {
    clear_error();
    if (validate_norm(p) != MORPHO_OK) return 0;
    DeviceInfo dev;
    const int sms = current_device_info(&dev) == MORPHO_OK ? dev.sms : 148;
    clear_error();
    return static_cast<size_t>(bwd_blocks(p->rows, p->dim, sms)) * 2 * p->dim * sizeof(float) + 256;
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
    const int blocks = bwd_blocks(p->rows, p->dim, dev.sms);
    const size_t need = static_cast<size_t>(blocks) * 2 * p->dim * sizeof(float);
    if (sums) {
        MORPHO_TRY(check_norm_ptr(workspace, "workspace", MORPHO_DTYPE_F32));
        if (workspace_bytes < need)
            return set_error(MORPHO_ERR_WORKSPACE, "layer norm workspace too small: %zu < %zu bytes", workspace_bytes, need);
    }
    NormArgs a = norm_args(p);
    a.x = h;
    a.w = weight;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.gy = grad_y;
    a.gh = grad_h;
    a.dx = dx;
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    const bool vec = p->dim * dtype_bytes(p->type) % 16 == 0 && rows_aligned(h, a.sx, p->type) &&
                     rows_aligned(grad_y, a.sgy, p->type) && rows_aligned(grad_h, a.sgh, p->type) && aligned16(dx);
    int rc;
    if (p->type == MORPHO_DTYPE_F16)
        rc = backward_t<__half>(a, vec, blocks, st);
    else if (p->type == MORPHO_DTYPE_BF16)
        rc = backward_t<__nv_bfloat16>(a, vec, blocks, st);
    else
        rc = backward_t<float>(a, vec, blocks, st);
    if (rc != MORPHO_OK || !sums) return rc;
    return reduce_partials(a, blocks, dweight, dbias, st);
}
