// grad_clip.cu -- the 2-norm over many gradients, and clipping by it (C ABI morpho_sm100_clip_grad_norm).
//   norm = sqrt(sum_i |g_i|^2) / loss_scale,   c = min(1, max_norm / (norm + 1e-6)) / loss_scale
//   out_i = c g_i
// Two passes over the gradients, bound by HBM: the first sums squares (fp32 within a thread, fp64
// between threads, blocks and tensors, always in the same order; a thread whose fp32 sum leaves its range
// takes its squares again in fp64), the second scales.  The norm is needed before anything can be written,
// so the second pass reads the gradients again, from L2 for what it still holds.  An infinite gradient makes
// the norm infinite and the factor zero: finite gradients become zero, infinite ones NaN (0 * inf); a NaN
// makes all of them NaN.
//
// The tensors are cut into chunks, dealt to a persistent grid, of one 2 KB segment for each warp.  The table
// of tensors travels as a kernel parameter, so a launch needs no copy to the device and can be captured in a
// graph.  Measured: 144 tensors, 65M fp16 values to fp32, 96 us (5.5 TB/s with the second read); 36 tensors of
// odd sizes, 7.2M bf16, 13 us in the kernels.  (Taking the chunks in reverse in the second pass, to
// find in L2 what the first read last, and storing with low cache priority changed nothing: 69 us each for 390 MB.)
//
// Alignment: a segment is read as the aligned 16-byte packs that cover it, with the neighbours' elements in
// the first and the last masked.  Where input and output stand differently to a 16-byte boundary the
// converted elements pass through shared memory, from which every aligned pack of the output is read as
// two packs and shifted together; only a segment's first and last few elements are stored one by one.
#include <algorithm>
#include <type_traits>

#include "elem.cuh"
#include "kernels.h"

namespace morpho {
namespace {

// A type of BYTES bytes (8 or 16) for one store.
template <size_t BYTES>
struct WordsOf {
    using type = uint4;
};
template <>
struct WordsOf<8> {
    using type = uint2;
};

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSegmentBytes = 2048;         // of one warp's input
constexpr int kSumPerSm = 8, kScalePerSm = 5;  // CTAs per SM
constexpr int kMaxBlocks = 2048;            // partial sums of one launch
constexpr int kTable = 768;                 // tensors per launch: the parameter block stays under 32 KB
constexpr int kFewTensors = 48, kSomeTensors = 192;  // smaller tables, cheaper to launch with

template <int N>
struct Table {
    int n, chunks;      // tensors; chunks in all
    int chunk0[N + 1];  // first chunk of each tensor
    const void* in[N];
    void* out[N];
    int64_t count[N];
    uint8_t in_type[N], out_type[N];
};
static_assert(sizeof(Table<kTable>) < 32000, "kernel parameter limit");

__host__ __device__ constexpr int segment_of(int type) { return kSegmentBytes / dtype_bytes(type); }  // elements
__host__ __device__ constexpr int chunk_of(int type) { return kWarps * segment_of(type); }

// The tensor that chunk `c` belongs to (the last one whose first chunk is not after it).
template <class Tab>
__device__ __forceinline__ int tensor_of(const Tab& t, int c) {
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

// f(pack, index of its first element) for the aligned packs of V elements that cover the warp's n elements
// from p on, of which `off` elements of the first belong to what stands before p.  A whole segment on a
// boundary has all its loads in flight at once.
template <int V, class T, class F>
__device__ __forceinline__ void each_pack(const T* p, int n, int off, F f) {
    constexpr int PACKS = kSegmentBytes / (V * sizeof(T)) / 32;
    const int lane = threadIdx.x & 31;
    if (off == 0 && n == kSegmentBytes / static_cast<int>(sizeof(T))) {
        Pack<T, V> x[PACKS];
#pragma unroll
        for (int i = 0; i < PACKS; ++i) x[i] = load_pack<T, V>(p + (i * 32 + lane) * V);
#pragma unroll
        for (int i = 0; i < PACKS; ++i) f(x[i], (i * 32 + lane) * V, std::true_type());
    } else {
#pragma unroll 2
        for (int e = lane * V - off; e < n; e += 32 * V) f(load_pack<T, V>(p + e), e, std::false_type());
    }
}

// A lane's fp32 sum of at most 32 squares is good between these: above, a square has overflowed; below, squares
// under 2^-126 have lost bits that count.  (fp16's squares stay far inside.)
constexpr float kLeastSum = 0x1p-100f, kMostSum = 0x1.fffffep127f;

template <class T>
__device__ __noinline__ double segment_squares_wide(const T* p, int n) {
    constexpr int V = 16 / sizeof(T);
    double s = 0.0;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
#pragma unroll 1
    for (int e = (threadIdx.x & 31) * V - off; e < n; e += 32 * V) {
        const Pack<T, V> x = load_pack<T, V>(p + e);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const double d = to_f32(x.v[k]);
            if (e + k >= 0 && e + k < n) s = fma(d, d, s);
        }
    }
    return s;
}

// This lane's share of the sum of squares of the warp's n elements from p on.
template <class T>
__device__ __forceinline__ double segment_squares(const T* p, int n) {
    constexpr int V = 16 / sizeof(T);
    float s = 0.f;
    uint32_t bits = 0u;  // of all elements: whether a sum of zero is one of zeros
    each_pack<V>(p, n, static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T)), [&](const auto& x, int e, auto whole) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (whole || (e + k >= 0 && e + k < n)) s = fmaf(to_f32(x.v[k]), to_f32(x.v[k]), s);
        if (!std::is_same<T, __half>::value) {
            const uint4 w = *reinterpret_cast<const uint4*>(x.v);
            bits |= w.x | w.y | w.z | w.w;
        }
    });
    constexpr uint32_t magnitude = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;  // (zeros of either sign are zeros)
    if (!std::is_same<T, __half>::value && (bits & magnitude) != 0u && !(s >= kLeastSum && s <= kMostSum)) return segment_squares_wide(p, n);
    return s;
}

template <class Tab>
__global__ void __launch_bounds__(kThreads, kSumPerSm) grad_squares_kernel(const __grid_constant__ Tab t, double* part) {
    __shared__ double scratch[kWarps];
    pdl_release();
    pdl_wait();
    double sum = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const int64_t at = static_cast<int64_t>(c - t.chunk0[i]) * chunk_of(t.in_type[i]) + (threadIdx.x >> 5) * segment_of(t.in_type[i]);
        const int n = static_cast<int>(min(static_cast<int64_t>(segment_of(t.in_type[i])), t.count[i] - at));
        if (n <= 0) continue;
        const int type = t.in_type[i];
        if (type == MORPHO_DTYPE_F32)
            sum += segment_squares(static_cast<const float*>(t.in[i]) + at, n);
        else if (type == MORPHO_DTYPE_F16)
            sum += segment_squares(static_cast<const __half*>(t.in[i]) + at, n);
        else
            sum += segment_squares(static_cast<const __nv_bfloat16*>(t.in[i]) + at, n);
    }
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// Four words of the 32 bytes a | b from byte `shift` (0..15) on.
__device__ __forceinline__ uint4 shift_packs(uint4 a, uint4 b, int shift) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (shift & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int bits = (shift & 3) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// q[0..n) = by * p[0..n) of one warp; `stage`: its shared memory, kStageBytes.
constexpr int kStageBytes = (segment_of(MORPHO_DTYPE_F16) + 16) * 4;

template <class T, class O>
__device__ __forceinline__ void segment_scale(const T* p, O* q, int n, float by, uint8_t* stage) {
    // as many elements as both sides move at once, so that a warp's stores cover whole sectors too
    constexpr int VO = 16 / sizeof(O), V = sizeof(T) > sizeof(O) ? 16 / sizeof(T) : VO;
    using Words = typename WordsOf<V * sizeof(O)>::type;
    const int lane = threadIdx.x & 31;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) % (V * sizeof(T)) / sizeof(T));
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(q) & 15u) / sizeof(O));
    auto scaled = [&](const auto& x) {
        Pack<O, V> y;
#pragma unroll
        for (int k = 0; k < V; ++k) y.v[k] = from_f32<O>(to_f32(x.v[k]) * by);
        return y;
    };
    if (mis % V == off) {  // packs fall on packs
        each_pack<V>(p, n, off, [&](const auto& x, int e, auto whole) {
            const Pack<O, V> y = scaled(x);
            if (whole || (e >= 0 && e + V <= n)) {
                *reinterpret_cast<Words*>(q + e) = *reinterpret_cast<const Words*>(y.v);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (e + k >= 0 && e + k < n) q[e + k] = y.v[k];
            }
        });
        return;
    }
    __syncwarp();  // the previous segment's packs have been read
    each_pack<V>(p, n, off, [&](const auto& x, int e, auto) {
        const Pack<O, V> y = scaled(x);
        *reinterpret_cast<Words*>(reinterpret_cast<O*>(stage) + e + off) = *reinterpret_cast<const Words*>(y.v);
    });
    __syncwarp();
    const int head = min(n, mis == 0 ? 0 : VO - mis);  // elements before q's first aligned pack
    const int packs = (n - head) / VO, tail = head + packs * VO;
    const O* from = reinterpret_cast<const O*>(stage) + off;
    const int byte0 = (off + head) * static_cast<int>(sizeof(O));
#pragma unroll 2
    for (int i = lane; i < packs; i += 32) {
        const uint4* a = reinterpret_cast<const uint4*>(stage) + (byte0 >> 4) + i;
        reinterpret_cast<uint4*>(q + head)[i] = shift_packs(a[0], a[1], byte0 & 15);
    }
    if (lane < head) q[lane] = from[lane];
    if (tail + lane < n) q[tail + lane] = from[tail + lane];
}

template <class Tab>
__global__ void __launch_bounds__(kThreads, kScalePerSm)
    grad_scale_kernel(const __grid_constant__ Tab t, const double* part, int parts, float max_norm, float loss_scale,
                      float* norm_out) {
    extern __shared__ __align__(16) uint8_t stages[];
    __shared__ double scratch[kWarps];
    pdl_release();
    pdl_wait();
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) sum += part[i];
    sum = block_sum(sum, scratch);
    // in fp64 to the factor itself, which is then one rounding away
    const double norm = sqrt(sum) / loss_scale;
    double c = max_norm / (norm + 1e-6);
    c = c > 1.0 ? 1.0 : c;  // NaN stays NaN
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
    const float by = static_cast<float>(c / loss_scale);
    uint8_t* stage = stages + (threadIdx.x >> 5) * kStageBytes;
    for (int k = blockIdx.x; k < t.chunks; k += gridDim.x) {
        const int i = tensor_of(t, k);
        const int64_t at = static_cast<int64_t>(k - t.chunk0[i]) * chunk_of(t.in_type[i]) + (threadIdx.x >> 5) * segment_of(t.in_type[i]);
        const int n = static_cast<int>(min(static_cast<int64_t>(segment_of(t.in_type[i])), t.count[i] - at));
        if (n <= 0 || (by == 1.0f && t.in[i] == t.out[i])) continue;  // in place and nothing to change
        auto out = [&](auto* p) {
            if (t.out_type[i] == MORPHO_DTYPE_F32)
                segment_scale(p + at, static_cast<float*>(t.out[i]) + at, n, by, stage);
            else if (t.out_type[i] == MORPHO_DTYPE_F16)
                segment_scale(p + at, static_cast<__half*>(t.out[i]) + at, n, by, stage);
            else
                segment_scale(p + at, static_cast<__nv_bfloat16*>(t.out[i]) + at, n, by, stage);
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
template <int N>
int64_t fill(Table<N>* t, const morpho_tensor_pair_t* pairs, int64_t first, int64_t count) {
    t->n = 0;
    int64_t chunks = 0, i = first;
    for (; i < count && t->n < N; ++i) {
        if (pairs[i].count == 0) continue;
        const int64_t more = (pairs[i].count + chunk_of(pairs[i].in_type) - 1) / chunk_of(pairs[i].in_type);
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

// Both passes, with tables of up to N tensors.
template <int N>
int clip(const DeviceInfo& dev, const morpho_tensor_pair_t* pairs, int64_t count, float max_norm, float loss_scale, float* norm, double* part,
         int64_t limit, cudaStream_t stream) {
    auto scale = grad_scale_kernel<Table<N>>;
    constexpr int smem = kWarps * kStageBytes;
    static_assert(smem <= 48 * 1024, "shared memory");
    Table<N> t;
    int launches = 0;
    int64_t parts = 0, i = 0;
    do {
        i = fill(&t, pairs, i, count);
        const int blocks = std::max(1, std::min({t.chunks, kSumPerSm * dev.sms, kMaxBlocks}));
        if (parts + blocks > limit) return set_error(MORPHO_ERR_WORKSPACE, "clip: too many elements for one call");
        prof_begin(stream, "grad_squares");
        MORPHO_CUDA_TRY(launch_after(grad_squares_kernel<Table<N>>, blocks, kThreads, 0, stream, t, part + parts));
        MORPHO_LAUNCH_CHECK("grad_squares");
        parts += blocks;
        ++launches;
    } while (i < count);
    i = 0;
    for (int k = 0; k < launches; ++k) {
        if (launches > 1) i = fill(&t, pairs, i, count);
        const int blocks = std::max(1, std::min(t.chunks, kScalePerSm * dev.sms));
        prof_begin(stream, "grad_scale");
        MORPHO_CUDA_TRY(launch_after(scale, blocks, kThreads, smem, stream, t, part, static_cast<int>(parts), max_norm, loss_scale, k == 0 ? norm : nullptr));
        MORPHO_LAUNCH_CHECK("grad_scale");
    }
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
    if (norm == nullptr || reinterpret_cast<uintptr_t>(norm) % sizeof(float) != 0)
        return set_error(MORPHO_ERR_INVALID, "clip: norm is NULL or not 4-byte aligned");
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return set_error(MORPHO_ERR_INVALID, "clip: workspace is NULL or not 16-byte aligned");
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    if (workspace_bytes < morpho_sm100_clip_grad_norm_workspace_size(count))
        return set_error(MORPHO_ERR_WORKSPACE, "clip workspace too small: %zu bytes", workspace_bytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* part = static_cast<double*>(workspace);
    const int64_t limit = static_cast<int64_t>(workspace_bytes / sizeof(double));
    return count <= kFewTensors    ? clip<kFewTensors>(dev, pairs, count, max_norm, loss_scale, norm, part, limit, st)
           : count <= kSomeTensors ? clip<kSomeTensors>(dev, pairs, count, max_norm, loss_scale, norm, part, limit, st)
                                   : clip<kTable>(dev, pairs, count, max_norm, loss_scale, norm, part, limit, st);
}
