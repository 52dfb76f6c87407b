// vocab_loss.cu -- softmax cross entropy of a linear layer over a large vocabulary, forward and
// backward, without keeping the logits (C ABI morpho_sm100_linear_cross_entropy_*).
//   z_tv = hidden_t . weight_v,   lse_t = log sum_v exp z_tv,   loss_t = lse_t - z_t,target(t)
//   dz_tv = g_t (exp(z_tv - lse_t) - [v = target(t)]),  dhidden = dz . weight,  dweight = dz^T . hidden
//
// Forward: one tcgen05 GEMM whose epilogue reduces each 128-column piece of a logit row in registers to
// its maximum and its sum of exponentials, so a [T, V] product leaves 16 bytes per row and 256 columns;
// a second kernel joins the pieces of a row in a fixed order.
// Backward: the vocabulary is taken in pieces of columns.  For each piece the logits are computed again
// (the same GEMM), turned into dz in the epilogue and written as a 16-bit [T, piece] matrix, which two
// GEMMs read: dhidden += dz . weight_piece (K = piece) and dweight_piece = dz^T . hidden (K = T, in
// pieces too).
// The arithmetic is 2TVD for the forward and 6TVD for the backward: the tensor cores bound it.
//
// dz is rounded to the inputs' type, as tcgen05 needs it, once, and before the common factor of the
// gradient is applied: with g_t = gmax r_t, |r_t| <= 1, the stored value is r_t (p - 1) 2^15 in fp16, so
// that probabilities down to 2^-29 stay normal numbers, and the epilogues multiply the fp32 sums by
// gmax 2^-15.  (bf16 has fp32's range and takes 2^0.)
//
// Warp roles of the GEMMs (320 threads): warp 0 TMA producer, warp 1 MMA issuer, warps 2-9 epilogue, as
// in the projection GEMM.
#include <algorithm>

#include "elem.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace morpho {
namespace {

constexpr uint32_t K_VOCAB = 6;  // kernel id in the device status word
constexpr int BM = 128, BN = 256, BK = 64;
constexpr int kGemmThreads = 320;
constexpr int kHalf = 128;  // columns an epilogue warp takes
constexpr int kStages = 4;
constexpr int kABytes = BM * BK * 2, kBBytes = BN * BK * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kBarOffset = kStages * kStageBytes;
constexpr int kSmemBytes = kBarOffset + 256 + 1024;

// A target that is neither in [0, vocab) nor ignore_index makes its row's lse NaN.
struct RowInfo {
    const int64_t* target;
    int64_t ignore_index;
    int vocab;
};

struct Gemm {
    int M, N;
    int k_blocks;
    int tiles_m, tiles_n;
    uint32_t* status;
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    return pack_half2(lo, hi);
}

// ---- epilogues: one thread per row, kHalf columns ---------------------------------------------

// Row statistics: the piece's maximum and sum of exp(z - maximum), and the target's logit.
struct EpiStats {
    struct Params {
        int64_t T;
        int V;
        const int64_t* target;
        float2* part;  // [ceil(V / 128)][T]
        float* zt;     // [T] logit of the target
    };
    __device__ static void run(const Params& p, uint32_t tacc, int64_t row, int n0) {
        const int64_t y = row < p.T ? p.target[row] : -1;
        float m = -INFINITY, s = 0.f, zt = 0.f;
#pragma unroll 1
        for (int cc = 0; cc < kHalf; cc += 32) {
            uint32_t r[32];
            tmem_ld32(tacc + cc, r);
            tmem_ld_wait();
            const int left = p.V - n0 - cc;  // live columns from here on
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i >= left) r[i] = __float_as_uint(-INFINITY);
                mx = fmaxf(mx, u2f(r[i]));
            }
            const float mn = fmaxf(m, mx);
            if (mn > -INFINITY) {
                const float b = mn * kLog2e;
                float t = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) t += ex2(fmaf(u2f(r[i]), kLog2e, -b));
                s = s * ex2(fmaf(m, kLog2e, -b)) + t;
                m = mn;
            } else {
                // -inf throughout, or NaN (which a maximum skips)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (u2f(r[i]) != u2f(r[i])) s = u2f(r[i]);
            }
            const int64_t at = y - n0 - cc;
            if (at >= 0 && at < 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i == at) zt = u2f(r[i]);
            }
        }
        if (row < p.T) {
            p.part[static_cast<int64_t>(n0 / kHalf) * p.T + row] = make_float2(m, s);
            if (y >= n0 && y < n0 + kHalf && y < p.V) p.zt[row] = zt;
        }
    }
};

// dz of one piece: r_t (exp(z - lse) - [v = target]), 16-bit.
template <bool BF16>
struct EpiDz {
    struct Params {
        int64_t T;
        int V, v0, ld;  // vocabulary; the piece's first column; row length of dz
        const int64_t* target;
        const float* lse;
        const float* row_scale;  // r_t 2^15 (0 for ignored rows)
        uint16_t* dz;            // [T, ld]
    };
    __device__ static void run(const Params& p, uint32_t tacc, int64_t row, int n0) {
        const bool live = row < p.T;
        const int64_t y = live ? p.target[row] : -1;
        const float l2 = live ? p.lse[row] * kLog2e : 0.f;
        const float rs = live ? p.row_scale[row] : 0.f;
#pragma unroll 1
        for (int cc = 0; cc < kHalf; cc += 32) {
            const int c0 = n0 + cc;  // column in the piece
            if (c0 >= p.ld) break;
            uint32_t r[32];
            tmem_ld32(tacc + cc, r);
            tmem_ld_wait();
            const int64_t at = y - p.v0 - c0;
            float d[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) d[i] = rs * ex2(fmaf(u2f(r[i]), kLog2e, -l2));
            if (at >= 0 && at < 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i == at) d[i] -= rs;
            }
            if (rs == 0.f) {  // an ignored row contributes nothing, whatever its logits are
#pragma unroll
                for (int i = 0; i < 32; ++i) d[i] = 0.f;
            }
            if (live) {
                uint4* dst = reinterpret_cast<uint4*>(p.dz + row * p.ld + c0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c0 + 8 * i < p.ld)
                        dst[i] = make_uint4(pack2<BF16>(d[8 * i], d[8 * i + 1]), pack2<BF16>(d[8 * i + 2], d[8 * i + 3]),
                                            pack2<BF16>(d[8 * i + 4], d[8 * i + 5]), pack2<BF16>(d[8 * i + 6], d[8 * i + 7]));
            }
        }
    }
};

// fp32 running sum over the pieces of K; the last one writes the scaled 16-bit result.
template <bool BF16>
struct EpiAcc {
    struct Params {
        int64_t M;
        int N;
        float* acc;  // [M, N]
        uint16_t* out;
        const float* scale;
        bool first, last;
    };
    __device__ static void run(const Params& p, uint32_t tacc, int64_t row, int n0) {
        const float g = *p.scale;
#pragma unroll 1
        for (int cc = 0; cc < kHalf; cc += 32) {
            if (n0 + cc >= p.N) break;
            uint32_t r[32];
            tmem_ld32(tacc + cc, r);
            tmem_ld_wait();
            if (row < p.M) {
                float4* acc = reinterpret_cast<float4*>(p.acc + row * p.N + n0 + cc);
                uint2* dst = reinterpret_cast<uint2*>(p.out + row * p.N + n0 + cc);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (n0 + cc + 4 * i < p.N) {
                        float4 x = make_float4(u2f(r[4 * i]), u2f(r[4 * i + 1]), u2f(r[4 * i + 2]), u2f(r[4 * i + 3]));
                        if (!p.first) {
                            const float4 o = acc[i];
                            x.x += o.x;
                            x.y += o.y;
                            x.z += o.z;
                            x.w += o.w;
                        }
                        if (p.last)
                            dst[i] = make_uint2(pack2<BF16>(g * x.x, g * x.y), pack2<BF16>(g * x.z, g * x.w));
                        else
                            acc[i] = x;
                    }
                }
            }
        }
    }
};

// ---- the GEMM -----------------------------------------------------------------------------------

// D (M x N) = A (M x K) B (K x N).  A_MN: A stored [K, M], else [M, K]; B_MN: B stored [K, N], else [N, K].
template <bool BF16, bool A_MN, bool B_MN, class Epi>
__global__ void __launch_bounds__(kGemmThreads, 1)
    vocab_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const int a_row0,
                      const int b_row0, const Gemm args, const typename Epi::Params ep) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOffset);
    constexpr int NB = 2 * kStages + 5;  // full, empty, acc_full[2], acc_empty[2], drain
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NB);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const int warp = warp_id();
    const int lane = threadIdx.x & 31;
    const int n_items = args.tiles_m * args.tiles_n;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + kStages);
    const uint32_t acc_full0 = smem_u32(bars + 2 * kStages), acc_empty0 = smem_u32(bars + 2 * kStages + 2);
    const uint32_t drain_bar = smem_u32(bars + 2 * kStages + 4);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full0 + 8 * a, 1);
            mbar_init(acc_empty0 + 8 * a, 8);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), 2 * BN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int g = 0;
            for (int w = blockIdx.x; w < n_items && !*abort_flag; w += gridDim.x) {
                const int m0 = (w / args.tiles_n) * BM, n0 = (w % args.tiles_n) * BN;
                for (int kb = 0; kb < args.k_blocks; ++kb, ++g) {
                    const int s = g % kStages;
                    if (g >= kStages && !mbar_wait(empty0 + 8 * s, ((g / kStages) & 1) ^ 1, args.status, K_VOCAB, 1)) {
                        *abort_flag = 1u;
                        break;
                    }
                    const uint32_t sA = smem_u32(smem + s * kStageBytes), sB = sA + kABytes, fb = full0 + 8 * s;
                    const int k0 = kb * BK;
                    mbar_arrive_expect_tx(fb, kStageBytes);
                    if (A_MN) {
                        tma_load_2d(sA, &tmA, fb, m0, a_row0 + k0);
                        tma_load_2d(sA + 64 * 128, &tmA, fb, m0 + 64, a_row0 + k0);
                    } else {
                        tma_load_2d(sA, &tmA, fb, k0, a_row0 + m0);
                    }
                    if (B_MN) {
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c) tma_load_2d(sB + c * 64 * 128, &tmB, fb, n0 + 64 * c, b_row0 + k0);
                    } else {
                        tma_load_2d(sB, &tmB, fb, k0, b_row0 + n0);
                    }
                }
            }
            if (*abort_flag)
                for (int i = max(0, g - kStages); i < g; ++i)
                    mbar_wait(full0 + 8 * (i % kStages), (i / kStages) & 1, args.status, K_VOCAB, 2);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = make_idesc_f16(BM, BN, A_MN, B_MN) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
        bool ok = true;
        int g = 0, j = 0;
        for (int w = blockIdx.x; ok && w < n_items; w += gridDim.x, ++j) {
            const int a = j & 1;
            if (j >= 2 && !mbar_wait_warp(acc_empty0 + 8 * a, ((j >> 1) & 1) ^ 1, args.status, K_VOCAB, 6)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t dacc = tmem + a * BN;
            for (int i = 0; i < args.k_blocks; ++i, ++g) {
                const int s = g % kStages;
                if (!mbar_wait_warp(full0 + 8 * s, (g / kStages) & 1, args.status, K_VOCAB, 3)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t sA = smem_u32(smem + s * kStageBytes), sB = sA + kABytes;
#pragma unroll
                for (int ks = 0; ks < BK / 16; ++ks) {
                    const uint64_t ad = A_MN ? make_sdesc(sA + ks * 2048, 64 * 128, 1024, SW_128) : make_sdesc(sA + ks * 32, 16, 1024, SW_128);
                    const uint64_t bd = B_MN ? make_sdesc(sB + ks * 2048, 64 * 128, 1024, SW_128) : make_sdesc(sB + ks * 32, 16, 1024, SW_128);
                    umma_ss_w(dacc, ad, bd, idesc, (i > 0 || ks > 0) ? 1u : 0u);
                }
                umma_commit_w(empty0 + 8 * s);
            }
            if (ok) umma_commit_w(acc_full0 + 8 * a);
        }
        if (!ok) {
            *abort_flag = 1u;
            umma_commit_w(drain_bar);
            mbar_wait_warp(drain_bar, 0, args.status, K_VOCAB, 4);
            umma_commit_w(acc_full0);
            umma_commit_w(acc_full0 + 8);
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
        int j = 0;
        for (int w = blockIdx.x; w < n_items; w += gridDim.x, ++j) {
            const int m0 = (w / args.tiles_n) * BM, n0 = (w % args.tiles_n) * BN;
            const int a = j & 1;
            if (!mbar_wait_warp(acc_full0 + 8 * a, (j >> 1) & 1, args.status, K_VOCAB, 5) || *abort_flag) {
                *abort_flag = 1u;
                break;
            }
            tc_fence_after();
            if (n0 + half * kHalf < args.N)
                Epi::run(ep, tmem + a * BN + half * kHalf + lane_off, static_cast<int64_t>(m0) + quad * 32 + lane, n0 + half * kHalf);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty0 + 8 * a);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * BN);
    }
}

// ---- small kernels ------------------------------------------------------------------------------

// Joins a row's pieces: lse = m + log(sum_i s_i exp(m_i - m)); loss = lse - z_target.  32 rows per block,
// eight threads a row.
__global__ void __launch_bounds__(256) vocab_join_kernel(const float2* part, int pieces, int64_t T, const float* zt,
                                                         RowInfo info, float* loss, float* lse) {
    __shared__ float2 sh[8][33];
    const int rx = threadIdx.x & 31, py = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + rx;
    float m = -INFINITY, s = 0.f;
    auto join = [&](float2 o) {
        const float mn = fmaxf(m, o.x);
        if (mn > -INFINITY) {
            s = s * expf(m - mn) + o.y * expf(o.x - mn);
            m = mn;
        } else {
            s += o.y;  // NaN, or nothing
        }
    };
    if (row < T)
        for (int i = py; i < pieces; i += 8) join(part[i * T + row]);
    sh[py][rx] = make_float2(m, s);
    __syncthreads();
    if (py != 0 || row >= T) return;
    for (int i = 1; i < 8; ++i) join(sh[i][rx]);
    const int64_t y = info.target[row];
    const bool ignored = y == info.ignore_index;
    float l = m + logf(s);
    if (!ignored && (y < 0 || y >= info.vocab)) l = NAN;
    lse[row] = l;
    loss[row] = ignored ? 0.f : l - zt[row];
}

__device__ __forceinline__ double block_total(double x, double* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    double r = 0.0;
    for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) r += scratch[i];
    __syncthreads();
    return r;
}

// One block: the sum or mean of the rows' losses.
__global__ void __launch_bounds__(1024) vocab_reduce_kernel(const float* rows, int64_t T, RowInfo info, bool mean,
                                                            float* out) {
    __shared__ double scratch[32];
    double sum = 0.0, kept = 0.0;
    for (int64_t i = threadIdx.x; i < T; i += 1024) {
        sum += rows[i];
        kept += info.target[i] != info.ignore_index ? 1.0 : 0.0;
    }
    sum = block_total(sum, scratch);
    kept = block_total(kept, scratch);
    if (threadIdx.x == 0) *out = static_cast<float>(mean ? sum / fmax(kept, 1.0) : sum);
}

// One block: splits the rows' gradients g_t into the factor that dz carries (row_scale = r_t unit) and
// the common one of the results (*common = gmax / unit).
__global__ void __launch_bounds__(1024) vocab_scale_kernel(const float* grad, int64_t T, RowInfo info, int reduction,
                                                           float unit, float* row_scale, float* common) {
    __shared__ double scratch[32];
    __shared__ float top[32];
    float most = 0.f;
    double kept = 0.0;
    for (int64_t i = threadIdx.x; i < T; i += 1024) {
        const bool keep = info.target[i] != info.ignore_index;
        kept += keep ? 1.0 : 0.0;
        if (keep && reduction == MORPHO_REDUCTION_NONE) {
            const float g = fabsf(grad[i]);
            most = isfinite(g) ? fmaxf(most, g) : most;
        }
    }
    kept = block_total(kept, scratch);
    if (reduction == MORPHO_REDUCTION_NONE) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = most;
        __syncthreads();
        for (int i = 0; i < 32; ++i) most = fmaxf(most, top[i]);
        if (most == 0.f) most = 1.f;
    } else {
        most = reduction == MORPHO_REDUCTION_MEAN ? static_cast<float>(*grad / fmax(kept, 1.0)) : *grad;
    }
    for (int64_t i = threadIdx.x; i < T; i += 1024) {
        const bool keep = info.target[i] != info.ignore_index;
        row_scale[i] = !keep ? 0.f : reduction == MORPHO_REDUCTION_NONE ? grad[i] / most * unit : unit;
    }
    if (threadIdx.x == 0) *common = most / unit;
}

// ---- host ---------------------------------------------------------------------------------------

constexpr size_t kPieceBytes = 512u << 20;  // dz of one piece of the vocabulary, at most
// Terms of one tensor-core sum, at most.  The tensor core truncates its fp32 accumulator at every
// K = 16 step, which biases a long sum towards zero (2.3e-8 of it a step; 1.2 % measured after 2^23
// terms), so longer sums are joined from sums of this length by rounded fp32 additions.
constexpr int kMaxK = 16384;

int validate_loss(const morpho_vocab_loss_t* p) {
    if (p == nullptr) return set_error(MORPHO_ERR_INVALID, "cross entropy problem is NULL");
    if (p->tokens < 0 || p->tokens > (1LL << 30)) return set_error(MORPHO_ERR_INVALID, "cross entropy: tokens = %lld out of range", static_cast<long long>(p->tokens));
    if (p->vocab <= 0 || p->vocab > (1 << 30)) return set_error(MORPHO_ERR_INVALID, "cross entropy: vocab = %d out of range", p->vocab);
    if (p->dim <= 0 || p->dim > kMaxK || p->dim % 8 != 0)
        return set_error(MORPHO_ERR_INVALID, "cross entropy: dim = %d must be a positive multiple of 8, at most %d", p->dim, kMaxK);
    if (p->type != MORPHO_DTYPE_F16 && p->type != MORPHO_DTYPE_BF16)
        return set_error(MORPHO_ERR_INVALID, "cross entropy: hidden and weight must be fp16 or bf16");
    if (p->reduction < MORPHO_REDUCTION_NONE || p->reduction > MORPHO_REDUCTION_SUM)
        return set_error(MORPHO_ERR_INVALID, "cross entropy: reduction %d unknown", p->reduction);
    for (const int64_t s : {p->stride_hidden, p->stride_weight})
        if (s != 0 && (s < p->dim || s % 8 != 0))
            return set_error(MORPHO_ERR_INVALID, "cross entropy: row stride %lld must be a multiple of 8 and at least dim", static_cast<long long>(s));
    return MORPHO_OK;
}

int64_t ld_hidden(const morpho_vocab_loss_t* p) { return p->stride_hidden ? p->stride_hidden : p->dim; }
int64_t ld_weight(const morpho_vocab_loss_t* p) { return p->stride_weight ? p->stride_weight : p->dim; }

// Columns of a vocabulary piece, a multiple of the tile width: as many as dz's limit and the length of a
// tensor-core sum allow.
int piece_cols(const morpho_vocab_loss_t* p) {
    const int64_t fit = static_cast<int64_t>(kPieceBytes / 2 / std::max<int64_t>(1, p->tokens)) / BN * BN;
    const int64_t all = (p->vocab + BN - 1) / BN * static_cast<int64_t>(BN);
    return static_cast<int>(std::min<int64_t>({all, std::max<int64_t>(BN, fit), kMaxK}));
}

struct Bump {
    uint8_t* base;
    size_t off = 0;
    template <class T>
    T* take(size_t count) {
        off = (off + 255) / 256 * 256;
        T* ptr = base ? reinterpret_cast<T*>(base + off) : nullptr;
        off += count * sizeof(T);
        return ptr;
    }
};

struct FwdPlan {
    float2* part;
    float *zt, *rows;
};
void plan_forward(Bump& b, const morpho_vocab_loss_t* p, FwdPlan* f) {
    const size_t T = p->tokens, pieces = (p->vocab + kHalf - 1) / kHalf;
    f->part = b.take<float2>(pieces * T);
    f->zt = b.take<float>(T);
    f->rows = b.take<float>(T);
}

struct BwdPlan {
    int cols;
    uint16_t* dz;
    float *row_scale, *common, *acc, *wacc;
};
void plan_backward(Bump& b, const morpho_vocab_loss_t* p, BwdPlan* f) {
    f->cols = piece_cols(p);
    f->dz = b.take<uint16_t>(static_cast<size_t>(p->tokens) * f->cols);
    f->row_scale = b.take<float>(p->tokens);
    f->common = b.take<float>(64);
    f->acc = b.take<float>(f->cols < p->vocab ? static_cast<size_t>(p->tokens) * p->dim : 0);
    f->wacc = b.take<float>(p->tokens > kMaxK ? static_cast<size_t>(f->cols) * p->dim : 0);
}

template <bool BF16, bool A_MN, bool B_MN, class Epi>
int run(const DeviceInfo& dev, const CUtensorMap& tA, const CUtensorMap& tB, int a_row0, int b_row0, int64_t M, int N, int64_t K,
        const typename Epi::Params& ep, cudaStream_t stream, const char* name) {
    auto kern = vocab_gemm_kernel<BF16, A_MN, B_MN, Epi>;
    MORPHO_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    Gemm g;
    g.M = static_cast<int>(M);
    g.N = N;
    g.k_blocks = static_cast<int>((K + BK - 1) / BK);
    g.tiles_m = static_cast<int>((M + BM - 1) / BM);
    g.tiles_n = (N + BN - 1) / BN;
    g.status = dev.status;
    const int64_t items = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
    if (items > 2147483647LL) return set_error(MORPHO_ERR_INVALID, "cross entropy: too many tiles");
    prof_begin(stream, name);
    kern<<<static_cast<unsigned>(std::min<int64_t>(items, dev.sms)), kGemmThreads, kSmemBytes, stream>>>(tA, tB, a_row0, b_row0, g, ep);
    MORPHO_LAUNCH_CHECK(name);
    return MORPHO_OK;
}

template <bool BF16>
int forward_t(const DeviceInfo& dev, const morpho_vocab_loss_t* p, const void* hidden, const void* weight,
              const RowInfo& info, float* loss, float* lse, const FwdPlan& f, cudaStream_t stream) {
    CUtensorMap tA, tB;
    MORPHO_TRY(make_tmap_2d_f16(&tA, hidden, p->tokens, p->dim, ld_hidden(p), BM, BK));
    MORPHO_TRY(make_tmap_2d_f16(&tB, weight, p->vocab, p->dim, ld_weight(p), BN, BK));
    EpiStats::Params ep{p->tokens, p->vocab, info.target, f.part, f.zt};
    MORPHO_TRY((run<BF16, false, false, EpiStats>(dev, tA, tB, 0, 0, p->tokens, p->vocab, p->dim, ep, stream, "vocab_stats")));
    const bool none = p->reduction == MORPHO_REDUCTION_NONE;
    prof_begin(stream, "vocab_join");
    vocab_join_kernel<<<static_cast<unsigned>((p->tokens + 31) / 32), 256, 0, stream>>>(
        f.part, (p->vocab + kHalf - 1) / kHalf, p->tokens, f.zt, info, none ? loss : f.rows, lse);
    MORPHO_LAUNCH_CHECK("vocab_join");
    if (!none) {
        prof_begin(stream, "vocab_reduce");
        vocab_reduce_kernel<<<1, 1024, 0, stream>>>(f.rows, p->tokens, info, p->reduction == MORPHO_REDUCTION_MEAN, loss);
        MORPHO_LAUNCH_CHECK("vocab_reduce");
    }
    return MORPHO_OK;
}

template <bool BF16>
int backward_t(const DeviceInfo& dev, const morpho_vocab_loss_t* p, const float* grad, const void* hidden, const void* weight,
               const RowInfo& info, const float* lse, void* dhidden, void* dweight, const BwdPlan& f, cudaStream_t stream) {
    prof_begin(stream, "vocab_scale");
    vocab_scale_kernel<<<1, 1024, 0, stream>>>(grad, p->tokens, info, p->reduction, BF16 ? 1.0f : 32768.0f, f.row_scale, f.common);
    MORPHO_LAUNCH_CHECK("vocab_scale");
    CUtensorMap tH, tW, tDz, tWn, tDzT, tHn;
    MORPHO_TRY(make_tmap_2d_f16(&tH, hidden, p->tokens, p->dim, ld_hidden(p), BM, BK));
    MORPHO_TRY(make_tmap_2d_f16(&tW, weight, p->vocab, p->dim, ld_weight(p), BN, BK));
    MORPHO_TRY(make_tmap_2d_f16(&tWn, weight, p->vocab, p->dim, ld_weight(p), BK, 64));
    MORPHO_TRY(make_tmap_2d_f16(&tHn, hidden, p->tokens, p->dim, ld_hidden(p), BK, 64));
    for (int v0 = 0; v0 < p->vocab; v0 += f.cols) {
        const int n = std::min(f.cols, p->vocab - v0);
        MORPHO_TRY(make_tmap_2d_f16(&tDz, f.dz, p->tokens, n, f.cols, BM, BK));
        MORPHO_TRY(make_tmap_2d_f16(&tDzT, f.dz, p->tokens, n, f.cols, BK, 64));
        typename EpiDz<BF16>::Params ez{p->tokens, p->vocab, v0, f.cols, info.target, lse, f.row_scale, f.dz};
        MORPHO_TRY((run<BF16, false, false, EpiDz<BF16>>(dev, tH, tW, 0, v0, p->tokens, n, p->dim, ez, stream, "vocab_dz")));
        typename EpiAcc<BF16>::Params ea{p->tokens, p->dim, f.acc, static_cast<uint16_t*>(dhidden), f.common, v0 == 0, v0 + n >= p->vocab};
        MORPHO_TRY((run<BF16, false, true, EpiAcc<BF16>>(dev, tDz, tWn, 0, v0, p->tokens, p->dim, n, ea, stream, "vocab_dhidden")));
        for (int64_t t0 = 0; t0 < p->tokens; t0 += kMaxK) {
            const int64_t k = std::min<int64_t>(kMaxK, p->tokens - t0);
            typename EpiAcc<BF16>::Params ew{n, p->dim, f.wacc, static_cast<uint16_t*>(dweight) + static_cast<int64_t>(v0) * p->dim,
                                             f.common, t0 == 0, t0 + k >= p->tokens};
            MORPHO_TRY((run<BF16, true, true, EpiAcc<BF16>>(dev, tDzT, tHn, static_cast<int>(t0), static_cast<int>(t0), n, p->dim, k, ew,
                                                            stream, "vocab_dweight")));
        }
    }
    return MORPHO_OK;
}

int check_loss_ptr(const void* p, const char* name, unsigned align) {
    if (p == nullptr) return set_error(MORPHO_ERR_INVALID, "cross entropy: %s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % align != 0) return set_error(MORPHO_ERR_INVALID, "cross entropy: %s is not %u-byte aligned", name, align);
    return MORPHO_OK;
}

}  // namespace
}  // namespace morpho

using namespace morpho;

extern "C" MORPHO_API size_t morpho_sm100_linear_cross_entropy_forward_workspace_size(const morpho_vocab_loss_t* p) {
    clear_error();
    if (validate_loss(p) != MORPHO_OK) return 0;
    Bump b{nullptr};
    FwdPlan f;
    plan_forward(b, p, &f);
    return b.off + 256;
}

extern "C" MORPHO_API size_t morpho_sm100_linear_cross_entropy_backward_workspace_size(const morpho_vocab_loss_t* p) {
    clear_error();
    if (validate_loss(p) != MORPHO_OK) return 0;
    Bump b{nullptr};
    BwdPlan f;
    plan_backward(b, p, &f);
    return b.off + 256;
}

extern "C" MORPHO_API int morpho_sm100_linear_cross_entropy_forward(const morpho_vocab_loss_t* p, const void* hidden,
                                                                    const void* weight, const int64_t* target, float* loss,
                                                                    float* lse, void* workspace, size_t workspace_bytes,
                                                                    void* stream) {
    const size_t need = morpho_sm100_linear_cross_entropy_forward_workspace_size(p);
    reset_launch_count();
    if (need == 0) return MORPHO_ERR_INVALID;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    MORPHO_TRY(check_loss_ptr(loss, "loss", p->tokens == 0 && p->reduction == MORPHO_REDUCTION_NONE ? 1 : 4));
    if (p->tokens == 0) {
        if (p->reduction != MORPHO_REDUCTION_NONE) MORPHO_CUDA_TRY(cudaMemsetAsync(loss, 0, sizeof(float), st));
        return MORPHO_OK;
    }
    MORPHO_TRY(check_loss_ptr(hidden, "hidden", 16));
    MORPHO_TRY(check_loss_ptr(weight, "weight", 16));
    MORPHO_TRY(check_loss_ptr(target, "target", 8));
    MORPHO_TRY(check_loss_ptr(lse, "lse", 4));
    MORPHO_TRY(check_loss_ptr(workspace, "workspace", 16));
    if (workspace_bytes < need) return set_error(MORPHO_ERR_WORKSPACE, "cross entropy workspace too small: %zu < %zu bytes", workspace_bytes, need);
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    Bump b{static_cast<uint8_t*>(workspace)};
    FwdPlan f;
    plan_forward(b, p, &f);
    const RowInfo info{target, p->ignore_index, p->vocab};
    return p->type == MORPHO_DTYPE_BF16 ? forward_t<true>(dev, p, hidden, weight, info, loss, lse, f, st)
                                        : forward_t<false>(dev, p, hidden, weight, info, loss, lse, f, st);
}

extern "C" MORPHO_API int morpho_sm100_linear_cross_entropy_backward(const morpho_vocab_loss_t* p, const float* grad_loss,
                                                                     const void* hidden, const void* weight,
                                                                     const int64_t* target, const float* lse, void* dhidden,
                                                                     void* dweight, void* workspace, size_t workspace_bytes,
                                                                     void* stream) {
    const size_t need = morpho_sm100_linear_cross_entropy_backward_workspace_size(p);
    reset_launch_count();
    if (need == 0) return MORPHO_ERR_INVALID;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    MORPHO_TRY(check_loss_ptr(dweight, "dweight", 16));
    if (p->tokens == 0) {
        MORPHO_CUDA_TRY(cudaMemsetAsync(dweight, 0, static_cast<size_t>(p->vocab) * p->dim * 2, st));
        return MORPHO_OK;
    }
    MORPHO_TRY(check_loss_ptr(grad_loss, "grad_loss", 4));
    MORPHO_TRY(check_loss_ptr(hidden, "hidden", 16));
    MORPHO_TRY(check_loss_ptr(weight, "weight", 16));
    MORPHO_TRY(check_loss_ptr(target, "target", 8));
    MORPHO_TRY(check_loss_ptr(lse, "lse", 4));
    MORPHO_TRY(check_loss_ptr(dhidden, "dhidden", 16));
    MORPHO_TRY(check_loss_ptr(workspace, "workspace", 16));
    if (workspace_bytes < need) return set_error(MORPHO_ERR_WORKSPACE, "cross entropy workspace too small: %zu < %zu bytes", workspace_bytes, need);
    DeviceInfo dev;
    MORPHO_TRY(current_device_info(&dev));
    Bump b{static_cast<uint8_t*>(workspace)};
    BwdPlan f;
    plan_backward(b, p, &f);
    const RowInfo info{target, p->ignore_index, p->vocab};
    return p->type == MORPHO_DTYPE_BF16 ? backward_t<true>(dev, p, grad_loss, hidden, weight, info, lse, dhidden, dweight, f, st)
                                        : backward_t<false>(dev, p, grad_loss, hidden, weight, info, lse, dhidden, dweight, f, st);
}
