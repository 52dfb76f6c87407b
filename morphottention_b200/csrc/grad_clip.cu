// grad_clip.cu -- the 2-norm over many gradients, and clipping by it (C ABI morpho_sm100_clip_grad_norm).
//   norm = sqrt(sum_i |g_i|^2) / loss_scale,   c = min(1, max_norm / (norm + 1e-6)) / loss_scale
//   out_i = c g_i
// Two passes over the gradients, bound by HBM: the first sums squares (fp32 within a thread, fp64
// between threads, blocks and tensors, always in the same order), the second scales.  The norm is
// needed before anything can be written, so the second pass reads the gradients again, from L2 for what
// it still holds.  A norm that is not finite makes the gradients non-finite (0 * inf, NaN), as dividing
// by it does.
//
// The tensors are cut into chunks of kChunk elements, dealt to a persistent grid; the table of tensors
// travels as a kernel parameter, so a launch needs no copy to the device and can be captured in a graph.
#include <algorithm>

#include "elem.cuh"
#include "kernels.h"

namespace morpho {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;      // elements
constexpr int kMaxBlocks = 1024;  // partial sums of one call
constexpr int kTable = 768;       // tensors per launch: the parameter block stays under 32 KB

struct Table {
    int n, chunks;          // tensors; chunks in all
    int chunk0[kTable + 1]; // first chunk of each tensor
    const void* in[kTable];
    void* out[kTable];
    int64_t count[kTable];
    uint8_t in_type[kTable], out_type[kTable];
};
static_assert(sizeof(Table) < 32000, "kernel parameter limit");

// The tensor that chunk `c` belongs to (the last one whose first chunk is not after it).
__device__ __forceinline__ int tensor_of(const Table& t, int c) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.chunk0[mid] <= c)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double x, double* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    double r = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) r += scratch[i];
    __syncthreads();
    return r;
}

template <class T>
__device__ __forceinline__ float chunk_squares(const T* p, int n) {
    float s = 0.f;
    constexpr int V = 16 / sizeof(T);
    if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        const int packs = n / V;
#pragma unroll 4
        for (int i = threadIdx.x; i < packs; i += kThreads) {
            const Pack<T, V> x = load_pack<T, V>(p + i * V);
#pragma unroll
            for (int k = 0; k < V; ++k) s = fmaf(to_f32(x.v[k]), to_f32(x.v[k]), s);
        }
        const int i = packs * V + threadIdx.x;
        if (i < n) s = fmaf(to_f32(p[i]), to_f32(p[i]), s);
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += kThreads) s = fmaf(to_f32(p[i]), to_f32(p[i]), s);
    }
    return s;
}

__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ Table t, double* part) {
    __shared__ double scratch[kThreads / 32];
    double sum = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const int64_t at = static_cast<int64_t>(c - t.chunk0[i]) * kChunk;
        const int n = static_cast<int>(min(static_cast<int64_t>(kChunk), t.count[i] - at));
        const int type = t.in_type[i];
        if (type == MORPHO_DTYPE_F32)
            sum += chunk_squares(static_cast<const float*>(t.in[i]) + at, n);
        else if (type == MORPHO_DTYPE_F16)
            sum += chunk_squares(static_cast<const __half*>(t.in[i]) + at, n);
        else
            sum += chunk_squares(static_cast<const __nv_bfloat16*>(t.in[i]) + at, n);
    }
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

template <class T, class O>
__device__ __forceinline__ void chunk_scale(const T* p, O* q, int n, float by) {
    constexpr int V = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
    const bool whole = reinterpret_cast<uintptr_t>(p) % (V * sizeof(T)) == 0 &&
                       reinterpret_cast<uintptr_t>(q) % (V * sizeof(O)) == 0;
    if (whole) {
        const int packs = n / V;
#pragma unroll 4
        for (int i = threadIdx.x; i < packs; i += kThreads) {
            const Pack<T, V> x = load_pack<T, V>(p + i * V);
            Pack<O, V> y;
#pragma unroll
            for (int k = 0; k < V; ++k) y.v[k] = from_f32<O>(to_f32(x.v[k]) * by);
            store_pack<O, V>(q + i * V, y);
        }
        const int i = packs * V + threadIdx.x;
        if (i < n) q[i] = from_f32<O>(to_f32(p[i]) * by);
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += kThreads) q[i] = from_f32<O>(to_f32(p[i]) * by);
    }
}

__global__ void __launch_bounds__(kThreads)
    grad_scale_kernel(const __grid_constant__ Table t, const double* part, int parts, float max_norm, float inv_scale,
                      float* norm_out) {
    __shared__ double scratch[kThreads / 32];
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) sum += part[i];
    sum = block_sum(sum, scratch);
    const float norm = static_cast<float>(sqrt(sum) * static_cast<double>(inv_scale));
    float c = max_norm / (norm + 1e-6f);
    c = c > 1.0f ? 1.0f : c;  // NaN stays NaN
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float by = c * inv_scale;
    for (int k = blockIdx.x; k < t.chunks; k += gridDim.x) {
        const int i = tensor_of(t, k);
        const int64_t at = static_cast<int64_t>(k - t.chunk0[i]) * kChunk;
        const int n = static_cast<int>(min(static_cast<int64_t>(kChunk), t.count[i] - at));
        if (by == 1.0f && t.in[i] == t.out[i]) continue;  // in place and nothing to change
        auto out = [&](auto* p) {
            if (t.out_type[i] == MORPHO_DTYPE_F32)
                chunk_scale(p + at, static_cast<float*>(t.out[i]) + at, n, by);
            else if (t.out_type[i] == MORPHO_DTYPE_F16)
                chunk_scale(p + at, static_cast<__half*>(t.out[i]) + at, n, by);
            else
                chunk_scale(p + at, static_cast<__nv_bfloat16*>(t.out[i]) + at, n, by);
        };
        if (t.in_type[i] == MORPHO_DTYPE_F32)
            out(static_cast<const float*>(t.in[i]));
        else if (t.in_type[i] == MORPHO_DTYPE_F16)
            out(static_cast<const __half*>(t.in[i]));
        else
            out(static_cast<const __nv_bfloat16*>(t.in[i]));
    }
}

// Fills the table from tensor `first` on; returns the tensor after the last one taken.
int64_t fill(Table* t, const morpho_tensor_pair_t* pairs, int64_t first, int64_t count) {
    t->n = 0;
    int64_t chunks = 0, i = first;
    for (; i < count && t->n < kTable; ++i) {
        if (pairs[i].count == 0) continue;
        const int64_t more = (pairs[i].count + kChunk - 1) / kChunk;
        if (chunks + more > (1LL << 30)) break;
        const int k = t->n++;
        t->chunk0[k] = static_cast<int>(chunks);
        t->in[k] = pairs[i].in;
        t->out[k] = pairs[i].out;
        t->count[k] = pairs[i].count;
        t->in_type[k] = static_cast<uint8_t>(pairs[i].in_type);
        t->out_type[k] = static_cast<uint8_t>(pairs[i].out_type);
        chunks += more;
    }
    t->chunks = static_cast<int>(chunks);
    t->chunk0[t->n] = t->chunks;
    return i;
}

int launch_squares(const Table& t, double* part, int blocks, cudaStream_t stream) {
    prof_begin(stream, "grad_squares");
    grad_squares_kernel<<<blocks, kThreads, 0, stream>>>(t, part);
    MORPHO_LAUNCH_CHECK("grad_squares");
    return MORPHO_OK;
}

int launch_scale(const Table& t, const double* part, int parts, float max_norm, float inv_scale, float* norm, int blocks,
                 cudaStream_t stream) {
    prof_begin(stream, "grad_scale");
    grad_scale_kernel<<<blocks, kThreads, 0, stream>>>(t, part, parts, max_norm, inv_scale, norm);
    MORPHO_LAUNCH_CHECK("grad_scale");
    return MORPHO_OK;
}

int validate_pairs(const morpho_tensor_pair_t* pairs, int64_t count) {
    if (count < 0 || (count > 0 && pairs == nullptr)) return set_error(MORPHO_ERR_INVALID, "clip: no tensors given");
    for (int64_t i = 0; i < count; ++i) {
        const morpho_tensor_pair_t& p = pairs[i];
        if (p.count < 0 || p.count > (1LL << 40))
            return set_error(MORPHO_ERR_INVALID, "clip: tensor %lld has %lld elements", static_cast<long long>(i), static_cast<long long>(p.count));
        if (p.in_type < MORPHO_DTYPE_F16 || p.in_type > MORPHO_DTYPE_F32 || p.out_type < MORPHO_DTYPE_F16 || p.out_type > MORPHO_DTYPE_F32)
            return set_error(MORPHO_ERR_INVALID, "clip: tensor %lld has an unknown element type", static_cast<long long>(i));
        if (p.count == 0) continue;
        if (p.in == nullptr || p.out == nullptr) return set_error(MORPHO_ERR_INVALID, "clip: tensor %lld is NULL", static_cast<long long>(i));
        if (reinterpret_cast<uintptr_t>(p.in) % dtype_bytes(p.in_type) != 0 || reinterpret_cast<uintptr_t>(p.out) % dtype_bytes(p.out_type) != 0)
            return set_error(MORPHO_ERR_INVALID, "clip: tensor %lld is not aligned to its element type", static_cast<long long>(i));
        if (p.in == p.out && p.in_type != p.out_type)
            return set_error(MORPHO_ERR_INVALID, "clip: tensor %lld is written in place with another type", static_cast<long long>(i));
    }
    return MORPHO_OK;
}

}  // namespace
}  // namespace morpho

using namespace morpho;

extern "C" MORPHO_API size_t morpho_sm100_clip_grad_norm_workspace_size(int64_t count) {
    // one fp64 partial per block of every launch of the first pass
    return count < 0 ? 0 : (static_cast<size_t>(count) / kTable + 2) * kMaxBlocks * sizeof(double) + 256;
}

extern "C" MORPHO_API int morpho_sm100_clip_grad_norm(const morpho_tensor_pair_t* pairs, int64_t count, float max_norm,
                                                      float loss_scale, float* norm, void* workspace,
                                                      size_t workspace_bytes, void* stream) {
    clear_error();
    reset_launch_count();
    MORPHO_TRY(validate_pairs(pairs, count));
    if (!(max_norm >= 0.0f)) return set_error(MORPHO_ERR_INVALID, "clip: max_norm must be non-negative (got %g)", static_cast<double>(max_norm));
    if (!(loss_scale > 0.0f) || loss_scale > 1e30f)
        return set_error(MORPHO_ERR_INVALID, "clip: loss_scale must be positive and finite (got %g)", static_cast<double>(loss_scale));
    if (norm == nullptr) return set_error(MORPHO_ERR_INVALID, "clip: norm is NULL");
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return set_error(MORPHO_ERR_INVALID, "clip: workspace is NULL or not 16-byte aligned");
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    if (workspace_bytes < morpho_sm100_clip_grad_norm_workspace_size(count))
        return set_error(MORPHO_ERR_WORKSPACE, "clip workspace too small: %zu bytes", workspace_bytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* part = static_cast<double*>(workspace);
    const float inv_scale = 1.0f / loss_scale;
    const int most = std::min(4 * dev.sms, kMaxBlocks);
    const int64_t limit = static_cast<int64_t>(workspace_bytes / sizeof(double));
    Table t;
    int launches = 0;
    int64_t parts = 0, i = 0;
    do {
        i = fill(&t, pairs, i, count);
        const int blocks = std::max(1, std::min(t.chunks, most));
        if (parts + blocks > limit) return set_error(MORPHO_ERR_WORKSPACE, "clip: too many elements for one call");
        MORPHO_TRY(launch_squares(t, part + parts, blocks, st));
        parts += blocks;
        ++launches;
    } while (i < count);
    i = 0;
    for (int k = 0; k < launches; ++k) {
        if (launches > 1) i = fill(&t, pairs, i, count);
        const int blocks = std::max(1, std::min(t.chunks, most));
        MORPHO_TRY(launch_scale(t, part, static_cast<int>(parts), max_norm, inv_scale, k == 0 ? norm : nullptr, blocks, st));
    }
    return MORPHO_OK;
}
