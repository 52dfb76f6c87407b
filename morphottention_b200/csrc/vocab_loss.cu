// vocab_loss.cu -- softmax cross entropy of a linear layer over a large vocabulary, forward and
// backward, without keeping the logits (C ABI morpho_sm100_linear_cross_entropy_*).
//   z_tv = hidden_t . weight_v,   lse_t = log sum_v exp z_tv,   loss_t = lse_t - z_t,target(t)
//   dz_tv = g_t (exp(z_tv - lse_t) - [v = target(t)]),  dhidden = dz . weight,  dweight = dz^T . hidden
//
// Forward: one tcgen05 GEMM whose epilogue reduces each 128-column piece of a logit row in registers to
// its maximum and its sum of exponentials, so a [T, V] product leaves 8 bytes per row and 128 columns;
// a second kernel joins the pieces of a row in a fixed order.
// Backward: the vocabulary is taken in pieces of columns.  For each piece the logits are computed again
// (the same GEMM), turned into dz in the epilogue and written as a 16-bit [T, piece] matrix, which two
// GEMMs read: dhidden += dz . weight_piece (K = piece) and dweight_piece = dz^T . hidden (K = T).
// The arithmetic is 2TVD for the forward and 6TVD for the backward: the tensor cores bound it.
//
// dz is rounded to the inputs' type, as tcgen05 needs it, once, and before the common factor of the
// gradient is applied: with g_t = gmax r_t, |r_t| <= 1, the stored value is r_t (p - 1) 2^15 in fp16, so
// that probabilities down to 2^-29 stay normal numbers, and the epilogues multiply the fp32 sums by
// gmax 2^-15.  (bf16 has fp32's range and takes 2^0.)
//
// The GEMMs run as 256 x 256 tiles of CTA pairs (cta_group::2): each SM reads half of A's rows and half of
// B's columns, 32 KB for every 64 of K, where a 128 x 256 tile of one CTA reads 48 KB and leaves its
// shared memory port busier than its tensor core.  Warp roles (608 threads): warp 0 TMA producer, warp 1
// MMA issuer (rank 0 of the pair), warps 2-17 epilogue, warp 18 scheduler; the accumulator is double-buffered in TMEM, and
// results leave through TMA stores from a swizzled box per warp.
//
// Measured, forward and backward (8TVD with the second logits; several B200s): 8192 tokens, 32768 x 512 fp16 1.02 to
// 1.06 ms, 1.04 to 1.08 PFLOP/s; 16384 tokens, 65536 x 1024 bf16 6.85 to 7.15 ms, 1.23 to 1.28 PFLOP/s, where the board's
// power limit holds a plain library product at 1.39.  256 tokens, 1000 x 256: 34 us, four dependent launches of 8 to 11,
// most of it each one's own set-up (608 threads, cluster barriers, TMEM) and one tile's serial load, product and epilogue.
// One token, 32768 x 1024, forward: 16.9 us, 67 MB read.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "elem.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace morpho {
namespace {

constexpr uint32_t K_VOCAB = 6;  // kernel id in the device status word
constexpr int kTile = 256;       // rows and columns of a CTA pair's tile
constexpr int kHalf = 128;       // rows of A, columns of B, and rows of the tile that one CTA holds
constexpr int BK = 128;          // K of a stage
constexpr int kEpiWarps = 16;    // two sets of eight, which take the tiles in turn: while one set's loads and
                                 // stores wait, the other's exponentials run
constexpr int kSetWarps = 8;
constexpr int kPiece = 128;      // columns of a tile that one warp takes,
constexpr int kLoad = 64;        // so many at once
constexpr int kGemmThreads = 32 * (kEpiWarps + 3);
constexpr int kStages = 3;
constexpr int kPanel = kHalf * 128;         // 16 KB: 128 rows of 128 bytes
constexpr int kOperandBytes = 2 * kPanel;   // 128 x 128 elements: two panels side by side
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kBoxBytes = 2048;                      // of an epilogue warp's stores: 32 rows of 64 bytes
constexpr int kStoreOffset = kStages * kStageBytes;  // a box for each of them
constexpr int kBarOffset = kStoreOffset + kEpiWarps * kBoxBytes;
constexpr int kBarBytes = 256;  // the barriers, then as much for the epilogue's sums
constexpr int kSmemBytes = kBarOffset + 2 * kBarBytes + 1024;
static_assert(kSmemBytes <= 232448, "shared memory");

// What a GEMM's epilogue does with its tile.
enum Kind : int {
    kStats,  // row statistics of the logits
    kDz,     // dz, 16-bit
    kOut,    // common * sum, 16-bit
    kPart,   // fp32 partial sums, one slab per K split
    kPartAdd // the same, added to what is there
};

// n / d for 0 <= n < 2^31 by one multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication"): mul is the low word of ceil(2^(32 + shift) / d), 2^shift the power of two not below d.
struct FastDiv {
    uint32_t mul, shift, d;
    static FastDiv of(int d) {
        FastDiv f{0, 0, static_cast<uint32_t>(d)};
        while ((1u << f.shift) < f.d) ++f.shift;
        f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - f.d)) / f.d + 1);
        return f;
    }
    __device__ __forceinline__ int div(int n) const {
        return static_cast<int>((__umulhi(mul, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> shift);
    }
};

// D (M x N) = A (M x K) B (K x N) as 256 x 256 tiles of CTA pairs, K cut into splits.
struct alignas(64) Task {
    CUtensorMap a, b, out;
    int kind;
    bool a_mn, b_mn;     // stored [K, M] / [K, N] (else [M, K] / [N, K])
    bool a_whole, b_whole;  // the map loads both panels of a stage at once (see load_map)
    int a_row0, b_row0;  // first row of A / B in its map
    int M, N;
    int tiles_m, tiles_n, group;  // `group` M tiles share each B tile in L2
    FastDiv by_slab, by_band, by_group, by_last;  // tiles; group x N tiles; group; M tiles of the last group
    int K, k_blocks, kb_per_split;
    int items_end;  // work items of this task and those before it
    int v0, padded; // kDz: the piece's first column of the vocabulary; its width in whole panels
    const uint8_t* dirty;  // per K block: whether B is read from Launch::clean instead (NULL: never)
};

// What the epilogues and the row kernels know of the rows.  A target that is neither in [0, V) nor
// ignore_index makes its row's lse NaN.
struct Rowwise {
    int64_t T;
    int V;
    const int64_t* target;
    int64_t ignore_index;
    int reduction;
    float unbias, log2e;  // what makes up for the tensor core's truncation of a logit (unbias_of), and log2(e) times it
    float2* part;   // forward: [pieces][T] maximum and sum of each piece of a row (kPiece columns, or a CTA's)
    float* zt;      // forward: [T] logit of the target
    uint32_t* done; // forward: the join kernel's count of finished blocks
    const float* lse;
    const float* grad;
    float unit, log2_unit;
    bool first;     // backward: this launch makes *common
    float* common;  // gmax / unit, the factor of the results; g_t = gmax r_t
};

// Rows that count for nothing (ignored, or of gradient zero) have zeros in dz, but dweight multiplies those by
// hidden, and padding may hold NaN or infinities there.  Such a row shows in its lse.  The first launch of a
// backward marks the blocks of BK rows that have one, and copies them with zeros in its place; dweight reads
// the copies of marked blocks and hidden itself for all others.  (Backward, every block marked: 256 x 1000 x 256 22 -> 43 us,
// 16384 x 1000 x 256 50 -> 77, 8192 x 32768 x 512 660 either way; none marked: 0.5 us at most.)
struct Clean {
    const uint16_t* hidden;
    int64_t ld;
    int D, blocks;
    uint16_t* copy;  // [T][D]
    uint8_t* dirty;  // [blocks]
};

constexpr int kMaxTasks = 3;
struct Launch {
    Task task[kMaxTasks];
    CUtensorMap clean;  // the copies
    Clean cleaning;     // of the first launch
    int tasks;
    Rowwise rows;
    uint32_t* next;  // work items taken after the first of each pair; NULL: dealt round-robin
    uint32_t* zero;  // counters of later launches to clear
    int zeros;
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

// ---- epilogues: one thread per row, kPiece columns at `tacc` ---------------------------------------

// Writes one box (32 rows of 64 bytes, this lane's row in `x`) to this warp's staging buffer in the TMA's
// 64-byte swizzle; lane 0 may then store it.
__device__ __forceinline__ void stage_box(uint32_t stage, int lane, const uint32_t* x) {
    if (lane == 0) bulk_wait_read_all();  // the previous box has left
    __syncwarp();
#pragma unroll
    for (int g = 0; g < 4; ++g)
        st_shared_u4(stage + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4), make_uint4(x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]));
    fence_proxy_async_smem();
    __syncwarp();
}

// f(registers, column) for the warp's columns of its 32 rows, kLoad at a time; `release` after the last load,
// when the accumulator may be written again.
template <class Release, class F>
__device__ __forceinline__ void each_load(uint32_t tacc, Release release, F f) {
#pragma unroll 1
    for (int c = 0; c < kPiece; c += kLoad) {
        uint32_t r[kLoad];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kLoad; i += 32) tmem_ld32(tacc + c + i, r + i);
        tmem_ld_wait();
        if (c + kLoad == kPiece) release();
        f(r, c);
    }
}

// Row statistics: the piece's maximum and sum of exp(z - maximum), and the target's logit.  Four
// independent chains each for the maximum and the sum.
template <class Release>
__device__ __forceinline__ void epi_stats(const Rowwise& p, uint32_t tacc, int64_t row, int n0, Release release) {
    const int64_t y = (row < p.T ? p.target[row] : -1) - n0;
    float m = -INFINITY, s = 0.f, zt = 0.f;
    each_load(tacc, release, [&](uint32_t* r, int c) {
        const int left = p.V - n0 - c;
        if (left < kLoad) {  // columns past the vocabulary
#pragma unroll
            for (int i = 0; i < kLoad; ++i)
                if (i >= left) r[i] = __float_as_uint(-INFINITY);
        }
        float m4[4], s4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m4[k] = u2f(r[k]);
            s4[k] = 0.f;
        }
#pragma unroll
        for (int i = 4; i + 8 <= kLoad; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) m4[k] = fmax3(m4[k], u2f(r[i + k]), u2f(r[i + 4 + k]));
#pragma unroll
        for (int k = 0; k < 4; ++k) m4[k] = fmaxf(m4[k], u2f(r[kLoad - 4 + k]));
        const float mn = fmaxf(m, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
        if (__any_sync(0xffffffffu, y >= c && y < c + kLoad)) {
#pragma unroll
            for (int i = 0; i < kLoad; ++i)
                if (c + i == y) zt = u2f(r[i]);
        }
        const float b = mn > -INFINITY ? mn * p.log2e : 0.f;  // -inf throughout, or NaN (which a maximum skips)
#pragma unroll
        for (int i = 0; i < kLoad; i += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) s4[k] += ex2(fmaf(u2f(r[i + k]), p.log2e, -b));
        s = s * ex2(fmaf(m, p.log2e, -b)) + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
        m = mn;
    });
    if (row < p.T) {
        p.part[static_cast<int64_t>(n0 / kPiece) * p.T + row] = make_float2(m * p.unbias, s);
        if (y >= 0 && y < kPiece && y + n0 < p.V) p.zt[row] = zt * p.unbias;
    }
}

// dz of one piece: r_t (exp(z - lse) - [v = target]) 2^15, the power of two in the exponent.
template <bool BF16, class Release>
__device__ __forceinline__ void epi_dz(const Rowwise& p, const Task& t, uint32_t tacc, int64_t row, int row0, int n0,
                                       uint32_t stage, int lane, float top, Release release) {
    const bool live = row < p.T;
    const int64_t target = live ? p.target[row] : -1;
    const int64_t y = target - t.v0 - n0;
    const float l2 = live ? p.lse[row] * kLog2e : 0.f;
    const bool own = p.reduction == MORPHO_REDUCTION_NONE;
    const float rt = !live || target == p.ignore_index ? 0.f : own ? p.grad[row] / top : 1.f;
    const float shift = p.log2_unit - l2;
    each_load(tacc, release, [&](uint32_t* r, int c) {
        const bool hit = __any_sync(0xffffffffu, y >= c && y < c + kLoad);
#pragma unroll
        for (int b = 0; b < kLoad; b += 32) {
            const int col = n0 + c + b;
            if (col < t.padded) {
                uint32_t* q = r + b;
#pragma unroll
                for (int i = 0; i < 32; ++i) q[i] = __float_as_uint(ex2(fmaf(u2f(q[i]), p.log2e, shift)));
                if (own) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) q[i] = __float_as_uint(rt * u2f(q[i]));
                }
                if (col + 32 > t.N) {  // columns past the piece, which are read as K: zeros
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (col + i >= t.N) q[i] = 0u;
                }
                if (hit) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + b + i == y) q[i] = __float_as_uint(fmaf(-rt, p.unit, u2f(q[i])));
                }
                uint32_t x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[i] = pack2<BF16>(u2f(q[2 * i]), u2f(q[2 * i + 1]));
                    if (rt == 0.f) x[i] = 0u;  // a row that counts for nothing adds nothing, whatever its logits are
                }
                stage_box(stage, lane, x);
                if (lane == 0) {
                    tma_store_2d(&t.out, stage, col, row0);
                    bulk_commit_group();
                }
            }
        }
    });
}

// 16-bit result: common * sum.
template <bool BF16, class Release>
__device__ __forceinline__ void epi_out(const Rowwise& p, const Task& t, uint32_t tacc, int row0, int n0, uint32_t stage,
                                        int lane, Release release) {
    const float g = *p.common;
    each_load(tacc, release, [&](uint32_t* r, int c) {
#pragma unroll
        for (int b = 0; b < kLoad; b += 32) {
            if (n0 + c + b < t.N) {
                uint32_t x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = pack2<BF16>(g * u2f(r[b + 2 * i]), g * u2f(r[b + 2 * i + 1]));
                stage_box(stage, lane, x);
                if (lane == 0) {
                    tma_store_2d(&t.out, stage, n0 + c + b, row0);
                    bulk_commit_group();
                }
            }
        }
    });
}

// fp32 partial sums of K split z.
template <class Release>
__device__ __forceinline__ void epi_part(const Task& t, uint32_t tacc, int row0, int n0, int z, uint32_t stage, int lane,
                                         Release release) {
    each_load(tacc, release, [&](uint32_t* r, int c) {
#pragma unroll
        for (int b = 0; b < kLoad; b += 16) {
            if (n0 + c + b < t.N) {
                stage_box(stage, lane, r + b);
                if (lane == 0) {
                    if (t.kind == kPartAdd)
                        tma_reduce_add_3d(&t.out, stage, n0 + c + b, row0, z);
                    else
                        tma_store_3d(&t.out, stage, n0 + c + b, row0, z);
                    bulk_commit_group();
                }
            }
        }
    });
}

// ---- the GEMM: up to three tasks in one persistent launch of CTA pairs -----------------------------

struct Item {
    int task, m0, n0, z;  // task -1: no more work
};

// Work item w: the tasks one after the other; within a task the splits, then groups of `group` M tiles,
// then the N tiles, then the M tiles of the group.
__device__ __forceinline__ Item item_of(const Launch& L, int w) {
    Item it{-1, 0, 0, 0};
    if (w >= L.task[L.tasks - 1].items_end) return it;
    int i = 0, start = 0;
    while (w >= L.task[i].items_end) start = L.task[i++].items_end;
    const Task& t = L.task[i];
    int r = w - start;
    it.task = i;
    it.z = t.by_slab.div(r);
    r -= it.z * static_cast<int>(t.by_slab.d);
    const int g = t.by_band.div(r);
    r -= g * static_cast<int>(t.by_band.d);
    const FastDiv& by = (g + 1) * t.group <= t.tiles_m ? t.by_group : t.by_last;
    const int n = by.div(r), gm = static_cast<int>(by.d);
    it.m0 = (g * t.group + r - n * gm) * kTile;
    it.n0 = n * kTile;
    return it;
}

__device__ __forceinline__ int first_block(const Task& t, const Item& it) { return it.z * t.kb_per_split; }
__device__ __forceinline__ int end_block(const Task& t, const Item& it) {
    return min(t.k_blocks, (it.z + 1) * t.kb_per_split);
}

// The items a CTA pair works on, published by rank 0's scheduler warp through a ring of kSlots in each CTA
// and read by the other roles in order.  The first item of a pair is its index, which all roles know.
// With two slots the scheduler takes an item when the epilogue has begun the last but one: early enough
// for the loads, late enough that pairs take the last items as they become free.
constexpr int kSlots = 2;
struct Items {
    uint32_t slot0, full0, empty0;  // shared-memory addresses: slots, full barriers; empty barriers (rank 0's)

    // The scheduler: item number n > 0.
    __device__ void publish(int n, const Item& it) const {
        const int s = n % kSlots;
        for (uint32_t r = 0; r < 2; ++r) {
            const uint32_t bar = cluster_addr(full0 + 8 * s, r);
            mbar_arrive_expect_tx_cluster(bar, 16);
            st_async_v4(cluster_addr(slot0 + 16 * s, r), bar, it.task, it.m0, it.n0, it.z);
        }
    }
    // Whether (in time) the slot for item n has been read by all.
    __device__ bool room(int n, uint32_t* status) const {
        return n <= kSlots || mbar_wait(empty0 + 8 * (n % kSlots), ((n - 1) / kSlots & 1) ^ 1, status, K_VOCAB, 8);
    }
    // Any other role: item number n > 0; false on a timeout.  One thread then calls taken(n).  Where the
    // items are dealt round-robin every role works them out for itself.
    __device__ bool read(int n, Item& it, const Launch& L, int first, int step) const {
        if (L.next == nullptr) {
            it = item_of(L, first + n * step);
            return true;
        }
        uint32_t* status = L.status;
        const int s = n % kSlots;
        if (!mbar_wait(full0 + 8 * s, ((n - 1) / kSlots) & 1, status, K_VOCAB, 9)) return false;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(it.task), "=r"(it.m0), "=r"(it.n0), "=r"(it.z)
                     : "r"(slot0 + 16 * s)
                     : "memory");
        return true;
    }
    __device__ void taken(int n, const Launch& L) const {
        if (L.next != nullptr) mbar_arrive_cluster(cluster_addr(empty0 + 8 * (n % kSlots), 0));
    }
};

// The largest finite |g_t| of the rows that are not ignored (1 if there is none), by the epilogue's threads.  At least
// unit x FLT_MIN, so that the later launches get the same value back from *common.
__device__ __forceinline__ float largest_gradient(const Rowwise& p, float* scratch, int thread) {
    float most = 0.f;
#pragma unroll 4
    for (int64_t i = thread; i < p.T; i += 32 * kEpiWarps) {
        const float g = fabsf(p.grad[i]);
        if (p.target[i] != p.ignore_index && isfinite(g)) most = fmaxf(most, g);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if ((thread & 31) == 0) scratch[thread >> 5] = most;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
#pragma unroll
    for (int i = 0; i < kEpiWarps; ++i) most = fmaxf(most, scratch[i]);
    return most > 0.f ? fmaxf(most, p.unit * FLT_MIN) : 1.f;
}

// Marks block `b` of rows and copies it if need be: one warp.
__device__ __forceinline__ void clean_block(const Rowwise& p, const Clean& c, int b, int lane) {
    const int64_t row0 = static_cast<int64_t>(b) * BK;
    uint32_t bad[BK / 32], any = 0u;
#pragma unroll
    for (int i = 0; i < BK / 32; ++i) {
        const int64_t row = row0 + 32 * i + lane;
        const bool out = row < p.T && !isfinite(p.lse[row]) &&
                         (p.target[row] == p.ignore_index || (p.reduction == MORPHO_REDUCTION_NONE && p.grad[row] == 0.f));
        bad[i] = __ballot_sync(0xffffffffu, out);
        any |= bad[i];
    }
    if (lane == 0) c.dirty[b] = any != 0u;
    if (any == 0u) return;
    const int rows = static_cast<int>(min(static_cast<int64_t>(BK), p.T - row0));
#pragma unroll
    for (int i = 0; i < BK / 32; ++i) {
        const int last = min(32, rows - 32 * i);
#pragma unroll 4
        for (int r = 0; r < last; ++r) {
            const int64_t row = row0 + 32 * i + r;
            for (int col = lane * 8; col < c.D; col += 256) {
                const uint4 x = *reinterpret_cast<const uint4*>(c.hidden + row * c.ld + col);
                *reinterpret_cast<uint4*>(c.copy + row * c.D + col) = bad[i] >> r & 1u ? make_uint4(0u, 0u, 0u, 0u) : x;
            }
        }
    }
    asm volatile("fence.proxy.async.global;" ::: "memory");  // the next launch reads it by TMA
}

// One operand of a stage: rows (M or N) x .. x + 127, K k .. k + 127, in two panels of 128 rows of 128 bytes.
// K-major: the panels are the halves of K; MN-major: the halves of the rows, each with K down.
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap& map, uint32_t bar, bool mn, bool whole, int row0,
                                             int x, int k) {
    if (mn) {
        if (whole) {
            tma_load_3d_pair(dst, &map, bar, 0, row0 + k, x / 64);
        } else {
            tma_load_2d_pair(dst, &map, bar, x, row0 + k);
            tma_load_2d_pair(dst + kPanel, &map, bar, x + 64, row0 + k);
        }
    } else if (whole) {
        tma_load_3d_pair(dst, &map, bar, 0, row0 + x, k / 64);
    } else {
        tma_load_2d_pair(dst, &map, bar, k, row0 + x);
        tma_load_2d_pair(dst + kPanel, &map, bar, k + 64, row0 + x);
    }
}

template <bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1) vocab_gemm_kernel(const __grid_constant__ Launch L) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOffset);
    // full, empty, acc_full[2], acc_empty[2], drain, item full, item empty
    constexpr int NB = 2 * kStages + 5 + 2 * kSlots;
    constexpr int kSlotWord = (NB * 8 + 8 + 15) / 16 * 4;  // first word of the item ring, after the two below
    static_assert(kSlotWord * 4 + 16 * kSlots <= kBarBytes, "barrier block");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NB);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const int warp = warp_id();
    const int lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    pdl_release();
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + kStages);
    const uint32_t acc_full0 = smem_u32(bars + 2 * kStages), acc_empty0 = smem_u32(bars + 2 * kStages + 2);
    const uint32_t drain_bar = smem_u32(bars + 2 * kStages + 4);
    const Items items{smem_u32(reinterpret_cast<uint32_t*>(bars) + kSlotWord), smem_u32(bars + 2 * kStages + 5), smem_u32(bars + 2 * kStages + 5 + kSlots)};
    if (threadIdx.x == 0) {
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(items.full0 + 8 * s, 1);    // rank 0's scheduler, to both
            mbar_init(items.empty0 + 8 * s, 3 + 2 * kSetWarps);  // used in rank 0: its MMA thread, both CTAs' producers and one set
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);   // used in rank 0: its producer's arrival and both CTAs' bytes
            mbar_init(empty0 + 8 * s, 1);  // rank 0's commit, to both
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full0 + 8 * a, 1);    // rank 0's commit, to both
            mbar_init(acc_empty0 + 8 * a, 2 * kSetWarps);  // used in rank 0: the buffer's epilogue set of both
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        fence_barrier_init();
        for (int i = 0; i < L.tasks; ++i) {
            tma_prefetch_desc(&L.task[i].a);
            tma_prefetch_desc(&L.task[i].b);
        }
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), 2 * kTile);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    if (L.rows.done != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *L.rows.done = 0u;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < L.zeros; i += kGemmThreads) L.zero[i] = 0u;

    if (warp == 0) {
        // ---------------- TMA producer, in both CTAs ----------------
        if (lane == 0) {
            int g = 0;
            Item it = item_of(L, first);
            for (int j = 0; !*abort_flag; ++j) {
                if (j > 0) {
                    if (!items.read(j, it, L, first, step)) {
                        *abort_flag = 1u;
                        break;
                    }
                    items.taken(j, L);
                }
                if (it.task < 0) break;
                const Task& t = L.task[it.task];
                const int kb0 = first_block(t, it), kb1 = end_block(t, it);
                const int m = it.m0 + rank * kHalf, n = it.n0 + rank * kHalf;
                uint32_t dirty = t.dirty != nullptr ? t.dirty[kb0] : 0u;
                for (int kb = kb0; kb < kb1; ++kb, ++g) {
                    const uint32_t dirty1 = t.dirty != nullptr && kb + 1 < kb1 ? t.dirty[kb + 1] : 0u;  // in flight beside this block
                    const int s = g % kStages;
                    if (g >= kStages && !mbar_wait(empty0 + 8 * s, ((g / kStages) & 1) ^ 1, L.status, K_VOCAB, 1)) {
                        *abort_flag = 1u;
                        break;
                    }
                    const uint32_t sA = smem_u32(smem + s * kStageBytes);
                    const uint32_t fb = cluster_addr(full0 + 8 * s, 0);
                    if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, 2 * kStageBytes);
                    load_operand(sA, t.a, fb, t.a_mn, t.a_whole, t.a_row0, m, kb * BK);
                    load_operand(sA + kOperandBytes, dirty ? L.clean : t.b, fb, t.b_mn, t.b_whole, t.b_row0, n, kb * BK);
                    dirty = dirty1;
                }
            }
            // No CTA leaves while commits to its barriers are on their way.
            for (int i = max(0, g - kStages); i < g && !*abort_flag; ++i)
                mbar_wait(empty0 + 8 * (i % kStages), (i / kStages) & 1, L.status, K_VOCAB, 7);
            // Drain: the loads of both CTAs complete on rank 0's barriers; rank 1 stays until the
            // cluster barrier at the end.
            if (*abort_flag && rank == 0)
                for (int i = max(0, g - kStages); i < g; ++i)
                    mbar_wait(full0 + 8 * (i % kStages), (i / kStages) & 1, L.status, K_VOCAB, 2);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer, one thread of rank 0 ----------------
        if (rank == 0 && lane == 0) {
            constexpr uint32_t type_bits = BF16 ? (1u << 7) | (1u << 10) : 0u;
            bool ok = true;
            int g = 0;
            Item it = item_of(L, first);
            for (int j = 0; ok && it.task >= 0; ++j) {
                const Task& t = L.task[it.task];
                const bool a_mn = t.a_mn, b_mn = t.b_mn;
                const int kb0 = first_block(t, it), kb1 = end_block(t, it);
                const uint32_t idesc = make_idesc_f16(kTile, kTile, a_mn, b_mn) | type_bits;
                const int a = j & 1;
                if (j >= 2 && !mbar_wait(acc_empty0 + 8 * a, ((j >> 1) & 1) ^ 1, L.status, K_VOCAB, 6)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t dacc = tmem + a * kTile;
                for (int kb = kb0; kb < kb1; ++kb, ++g) {
                    const int s = g % kStages;
                    // (what the TMA wrote needs no tcgen05 fence: the MMAs read it through the async proxy)
                    if (!mbar_wait(full0 + 8 * s, (g / kStages) & 1, L.status, K_VOCAB, 3)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sA = smem_u32(smem + s * kStageBytes), sB = sA + kOperandBytes;
                    const int left = t.K - kb * BK;  // the last stage may hold less: whole K = 16 steps of zeros are left out
#pragma unroll
                    for (int ks = 0; ks < BK / 16; ++ks) {
                        // K-major: K = 16 every 32 bytes of a panel's rows, 8-row groups of 1 KB; MN-major:
                        // K = 16 every 2 KB, the second 64 rows a panel further
                        const uint32_t kmaj = (ks / 4) * kPanel + (ks % 4) * 32, mnmaj = ks * 2048;
                        if (ks * 16 < left)
                            umma_ss_pair(dacc, make_sdesc(sA + (a_mn ? mnmaj : kmaj), a_mn ? kPanel : 16, 1024, SW_128),
                                         make_sdesc(sB + (b_mn ? mnmaj : kmaj), b_mn ? kPanel : 16, 1024, SW_128), idesc,
                                         (kb > kb0 || ks > 0) ? 1u : 0u);
                    }
                    umma_commit_pair(empty0 + 8 * s);
                }
                if (ok) umma_commit_pair(acc_full0 + 8 * a);
                if (ok && !items.read(j + 1, it, L, first, step)) ok = false;
                if (ok) items.taken(j + 1, L);
            }
            if (!ok) {
                *abort_flag = 1u;
                umma_commit_pair(drain_bar);
                mbar_wait(drain_bar, 0, L.status, K_VOCAB, 4);
                umma_commit_pair(acc_full0);
                umma_commit_pair(acc_full0 + 8);
            }
        }
        // One warp counts the rows of a mean for the launches that scale results by it, beside the tiles.  With many
        // tokens and a small vocabulary it takes longer than they do: backward of 2^20 tokens, 300 x 64, 2.97 ms where a
        // sum takes 1.06; 16384 tokens, 1000 x 256, 51.5 us and 50.0; 8192, 32768 x 512, no difference.
        if (blockIdx.x == 1 && L.rows.first && L.rows.reduction != MORPHO_REDUCTION_NONE) {
            int64_t kept = 0;
            if (L.rows.reduction == MORPHO_REDUCTION_MEAN) {
#pragma unroll 8
                for (int64_t i = lane; i < L.rows.T; i += 32) kept += L.rows.target[i] != L.rows.ignore_index;
                for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, o);
            }
            if (lane == 0) *L.rows.common = *L.rows.grad / (static_cast<float>(max(kept, int64_t(1))) * L.rows.unit);
        }
    } else if (warp == kEpiWarps + 2) {
        // ---------------- scheduler, one thread of rank 0 (and, in a backward's first launch, the rows that count for nothing) ----
        if (L.rows.first)
            for (int b = blockIdx.x; b < L.cleaning.blocks; b += gridDim.x) clean_block(L.rows, L.cleaning, b, lane);
        if (rank == 0 && lane == 0 && L.next != nullptr) {
            Item it = item_of(L, first);
            // the end is published twice: each epilogue set reads every other item
            for (int j = 1, ends = it.task < 0; ends < 2; ++j) {
                if (!items.room(j, L.status)) {
                    *abort_flag = 1u;
                    break;
                }
                if (ends == 0) it = item_of(L, step + static_cast<int>(atomicAdd(L.next, 1u)));
                ends += it.task < 0;
                items.publish(j, it);
            }
        }
    } else {
        // ---------------- epilogue, in both CTAs ----------------
        const int set = (warp - 2) / kSetWarps, quad = warp & 3, piece = ((warp - 2) >> 2) & 1;
        const uint32_t stage = smem_u32(smem + kStoreOffset + (warp - 2) * kBoxBytes);
        // Per-token gradients: the largest of them.  The first launch looks for itself, in every CTA (a few us
        // beside the first tile's loads), and leaves it to the others.
        float top = 1.f;
        if (L.rows.reduction == MORPHO_REDUCTION_NONE && L.rows.grad != nullptr) {
            if (L.rows.first) {
                top = largest_gradient(L.rows, reinterpret_cast<float*>(smem + kBarOffset + kBarBytes), threadIdx.x - 64);
                if (blockIdx.x == 0 && threadIdx.x == 64) *L.rows.common = top / L.rows.unit;
            } else {
                top = *L.rows.common * L.rows.unit;
            }
        }
        Item it = item_of(L, first);
        for (int j = set;; j += 2) {  // set 0 the even items, set 1 the odd ones
            if (j > 0) {
                const bool ok = items.read(j, it, L, first, step);
                if (!__all_sync(0xffffffffu, ok)) {
                    *abort_flag = 1u;
                    break;
                }
                if (lane == 0) items.taken(j, L);
            }
            if (it.task < 0) break;
            const Task& t = L.task[it.task];
            const int a = j & 1;
            if (!mbar_wait_warp(acc_full0 + 8 * a, (j >> 1) & 1, L.status, K_VOCAB, 5) || *abort_flag) {
                *abort_flag = 1u;
                break;
            }
            tc_fence_after();
            const int row0 = it.m0 + rank * kHalf + quad * 32, n0 = it.n0 + piece * kPiece;
            const uint32_t tacc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + a * kTile + piece * kPiece;
            auto release = [&]() {  // this warp has read its part of the accumulator
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(cluster_addr(acc_empty0 + 8 * a, 0));
            };
            if (n0 >= t.N || row0 >= t.M) {  // (dz: its padding ends inside the last live piece)
                release();
            } else if (t.kind == kStats) {
                epi_stats(L.rows, tacc, static_cast<int64_t>(row0) + lane, n0, release);
            } else if (t.kind == kDz) {
                epi_dz<BF16>(L.rows, t, tacc, static_cast<int64_t>(row0) + lane, row0, n0, stage, lane, top, release);
            } else if (t.kind == kOut) {
                epi_out<BF16>(L.rows, t, tacc, row0, n0, stage, lane, release);
            } else {
                epi_part(t, tacc, row0, n0, it.z, stage, lane, release);
            }
        }
        if (lane == 0) bulk_wait_all();  // the stores have read this CTA's shared memory and are done
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 2 * kTile);
    }
}

// out = common * sum of the partial slabs (in their order): 16-bit, eight elements a thread.
template <bool BF16>
__global__ void __launch_bounds__(256) vocab_finish_kernel(const float* part, int slabs, int64_t elems, const float* common,
                                                           uint16_t* out) {
    pdl_release();
    pdl_wait();
    const float g = *common;
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < elems; i += static_cast<int64_t>(gridDim.x) * 2048) {
        float4 a = *reinterpret_cast<const float4*>(part + i), b = *reinterpret_cast<const float4*>(part + i + 4);
        for (int s = 1; s < slabs; ++s) {
            const float4 c = *reinterpret_cast<const float4*>(part + s * elems + i), d = *reinterpret_cast<const float4*>(part + s * elems + i + 4);
            a.x += c.x, a.y += c.y, a.z += c.z, a.w += c.w;
            b.x += d.x, b.y += d.y, b.z += d.z, b.w += d.w;
        }
        *reinterpret_cast<uint4*>(out + i) = make_uint4(pack2<BF16>(g * a.x, g * a.y), pack2<BF16>(g * a.z, g * a.w),
                                                        pack2<BF16>(g * b.x, g * b.y), pack2<BF16>(g * b.z, g * b.w));
    }
}

// ---- a few tokens: logits on CUDA cores ------------------------------------------------------------

constexpr int kFewTokens = 2;  // (32768 x 1024: 16 and 19 us; with three or four 26, and the tensor cores take 25 for any number up to 256)
constexpr int kFewWarps = 8;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kFewMaxStages = 6, kFewRing = 192 * 1024;
constexpr int kFewMaxDim = 6144;  // two stages for every warp in the ring

// (m, s) <- (m, s) joined with (om, os): m the maximum, s the sum of exp(z - m).
__device__ __forceinline__ void join(float& m, float& s, float om, float os) {
    const float mn = fmaxf(m, om);
    if (mn > -INFINITY) {
        s = s * ex2((m - mn) * kLog2e) + os * ex2((om - mn) * kLog2e);
        m = mn;
    } else {
        s += os;  // NaN, or nothing
    }
}

template <bool BF16>
__device__ __forceinline__ void unpack8(uint4 x, float* f) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (BF16) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
}

// Up to TT tokens against the whole vocabulary, bound by reading the weight once.  Each warp streams a
// contiguous range of rows through a ring of its own in shared memory (bulk copies of R 32 / GL rows), so the
// bytes in flight do not hang on registers; GL lanes share R rows, the groups of a warp work on as many, each
// keeping the running maximum and sum of its own.  The hidden rows stand in shared memory too, and every
// CTA (one per SM) leaves one piece of each token's statistics.
template <bool BF16, int TT, int GL, int R>
__global__ void __launch_bounds__(kFewThreads, 1) vocab_few_kernel(const Rowwise p, const uint16_t* hidden, int64_t ldh, const uint16_t* weight,
                                                                   int64_t ldw, int D, int stages, uint32_t* status) {
    constexpr int GROUPS = 32 / GL, ROWS = R * GROUPS;  // rows at a time: g, g + GROUPS of every stage
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t bars[kFewWarps * kFewMaxStages];
    __shared__ float2 sh[kFewWarps][TT];
    const int lane = threadIdx.x & 31, warp = warp_id(), l = lane % GL, g = lane / GL;
    const int T = static_cast<int>(p.T), chunks = D / 8, row_bytes = 2 * D, stage_bytes = ROWS * row_bytes;
    uint4* hs = reinterpret_cast<uint4*>(ring + kFewWarps * stages * stage_bytes);  // [TT][D / 8]
    const uint8_t* mine = ring + warp * stages * stage_bytes;
    const uint32_t bar0 = smem_u32(bars + warp * kFewMaxStages);
    pdl_release();
    if (lane < kFewMaxStages) mbar_init(bar0 + 8 * lane, 1);
    fence_barrier_init();
    __syncwarp();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0u;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kFewWarps, per = (p.V + warps - 1) / warps;
    const int v0 = static_cast<int>(min(static_cast<int64_t>(p.V), (static_cast<int64_t>(blockIdx.x) * kFewWarps + warp) * per));
    const int n = static_cast<int>(min(static_cast<int64_t>(p.V) - v0, per));  // this warp's rows
    auto fetch = [&](int i) {
        const int rows = min(ROWS, n - i * ROWS);
        if (rows <= 0) return;
        const uint32_t bar = bar0 + 8 * (i % stages), dst = smem_u32(mine + (i % stages) * stage_bytes);
        const uint16_t* src = weight + (static_cast<int64_t>(v0) + i * ROWS) * ldw;
        mbar_arrive_expect_tx(bar, rows * row_bytes);
        if (ldw == D) {
            bulk_load(dst, src, rows * row_bytes, bar);
        } else {
            for (int r = 0; r < rows; ++r) bulk_load(dst + r * row_bytes, src + r * ldw, row_bytes, bar);
        }
    };
    if (lane == 0)
        for (int i = 0; i < stages; ++i) fetch(i);
    for (int i = threadIdx.x; i < TT * chunks; i += kFewThreads) {
        const int t = i / chunks;
        hs[i] = t < T ? *reinterpret_cast<const uint4*>(hidden + t * ldh + (i - t * chunks) * 8) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    int64_t y[TT];
    float m[TT], s[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        y[t] = t < T ? p.target[t] - v0 : -1;
        m[t] = -INFINITY;
        s[t] = 0.f;
    }
    for (int i = 0; i * ROWS < n; ++i) {
        if (!mbar_wait_warp(bar0 + 8 * (i % stages), (i / stages) & 1, status, K_VOCAB, 10)) {
            for (int k = i + 1; k < i + stages && k * ROWS < n; ++k)  // the copies in flight
                mbar_wait_warp(bar0 + 8 * (k % stages), (k / stages) & 1, status, K_VOCAB, 11);
            break;
        }
        const uint4* row = reinterpret_cast<const uint4*>(mine + (i % stages) * stage_bytes + g * row_bytes);
        float acc[R][TT][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[r][t][0] = acc[r][t][1] = 0.f;
#pragma unroll 2
        for (int c = l; c < chunks; c += GL) {
            float f[R][8];
#pragma unroll
            for (int r = 0; r < R; ++r) unpack8<BF16>(row[r * GROUPS * chunks + c], f[r]);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                float h[8];
                unpack8<BF16>(hs[t * chunks + c], h);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[r][t][k & 1] = fmaf(f[r][k], h[k], acc[r][t][k & 1]);
            }
        }
        __syncwarp();
        if (lane == 0) fetch(i + stages);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int q = i * ROWS + r * GROUPS + g;
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                float z = acc[r][t][0] + acc[r][t][1];
#pragma unroll
                for (int o = GL / 2; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
                if (q < n) {  // (a short last stage holds older rows past it)
                    join(m[t], s[t], z, z == z ? 1.f : z);
                    if (l == 0 && y[t] == q) p.zt[t] = z;
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
        for (int o = GL; o < 32; o <<= 1) join(m[t], s[t], __shfl_xor_sync(0xffffffffu, m[t], o), __shfl_xor_sync(0xffffffffu, s[t], o));
        if (lane == 0) sh[warp][t] = make_float2(m[t], s[t]);
    }
    __syncthreads();
    if (threadIdx.x < T) {
        const int t = threadIdx.x;
        float mm = -INFINITY, ss = 0.f;
        for (int i = 0; i < kFewWarps; ++i) join(mm, ss, sh[i][t].x, sh[i][t].y);
        p.part[static_cast<int64_t>(blockIdx.x) * T + t] = make_float2(mm, ss);
    }
}

// ---- row kernels ------------------------------------------------------------------------------------

constexpr int kJoinThreads = 256;

// Joins a row's pieces: lse = m + log(sum_i s_i exp(m_i - m)); loss = lse - z_target.  R rows a block,
// kJoinThreads / R threads a row, in a fixed order.  For a sum or a mean, each block leaves its rows'
// sum and the block that ends last adds those up, again in a fixed order.
template <int R>
__global__ void __launch_bounds__(kJoinThreads) vocab_join_kernel(const Rowwise p, int pieces, double2* block_sums, float* loss, float* lse) {
    constexpr int P = kJoinThreads / R;
    __shared__ float2 sh[kJoinThreads];
    __shared__ double2 sums[kJoinThreads / 32];
    __shared__ bool last;
    pdl_release();
    pdl_wait();
    const int rx = threadIdx.x % R, py = threadIdx.x / R;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * R + rx;
    float m = -INFINITY, s = 0.f;
    if (row < p.T) {
        int i = py;
        for (; i + 3 * P < pieces; i += 4 * P) {
            float2 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = p.part[(static_cast<int64_t>(i) + k * P) * p.T + row];
#pragma unroll
            for (int k = 0; k < 4; ++k) join(m, s, o[k].x, o[k].y);
        }
        for (; i < pieces; i += P) {
            const float2 o = p.part[static_cast<int64_t>(i) * p.T + row];
            join(m, s, o.x, o.y);
        }
    }
    sh[threadIdx.x] = make_float2(m, s);
#pragma unroll
    for (int n = P / 2; n > 0; n >>= 1) {
        __syncthreads();
        if (py < n) {
            const float2 o = sh[threadIdx.x + n * R];
            join(m, s, o.x, o.y);
            sh[threadIdx.x] = make_float2(m, s);
        }
    }
    double l = 0.0, kept = 0.0;
    if (py == 0 && row < p.T) {
        const int64_t y = p.target[row];
        const bool ignored = y == p.ignore_index;
        float e = m + logf(s);
        if (!ignored && (y < 0 || y >= p.V)) e = NAN;
        lse[row] = e;
        const float one = ignored ? 0.f : e - p.zt[row];
        if (p.reduction == MORPHO_REDUCTION_NONE) loss[row] = one;
        l = one;
        kept = ignored ? 0.0 : 1.0;
    }
    if (p.reduction == MORPHO_REDUCTION_NONE) return;
    auto block_sum = [&]() {  // into thread 0
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
            kept += __shfl_xor_sync(0xffffffffu, kept, o);
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = make_double2(l, kept);
        __syncthreads();
        if (threadIdx.x == 0)
            for (int i = 1; i < kJoinThreads / 32; ++i) {
                l += sums[i].x;
                kept += sums[i].y;
            }
    };
    block_sum();
    if (threadIdx.x == 0) {
        block_sums[blockIdx.x] = make_double2(l, kept);
        __threadfence();
        last = atomicAdd(p.done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    l = kept = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kJoinThreads) {
        const double2 o = __ldcg(block_sums + i);
        l += o.x;
        kept += o.y;
    }
    block_sum();
    if (threadIdx.x == 0) *loss = static_cast<float>(p.reduction == MORPHO_REDUCTION_MEAN ? l / fmax(kept, 1.0) : l);
}

// ---- host ---------------------------------------------------------------------------------------

constexpr size_t kPieceBytes = 512u << 20;  // dz of one piece of the vocabulary, at most; two are held
// Terms of one tensor-core sum, at most.  The tensor core truncates its fp32 accumulator at every
// K = 16 step, which biases a long sum towards zero (2.3e-8 of it a step; 1.2 % measured after 2^23
// terms), so longer sums are joined from sums of this length by rounded fp32 additions.  What that leaves in
// dhidden and dweight, up to 5e-5 of a sum, is a tenth of the most that rounding the result to fp16 costs; the
// logits, which are not rounded, are corrected instead (unbias_of).
constexpr int kMaxK = 32768;
constexpr int kMaxDim = 16384;

int validate_loss(const morpho_vocab_loss_t* p) {
    if (p == nullptr) return set_error(MORPHO_ERR_INVALID, "cross entropy problem is NULL");
    if (p->tokens < 0 || p->tokens > (1LL << 30)) return set_error(MORPHO_ERR_INVALID, "cross entropy: tokens = %lld out of range", static_cast<long long>(p->tokens));
    if (p->vocab <= 0 || p->vocab > (1 << 30)) return set_error(MORPHO_ERR_INVALID, "cross entropy: vocab = %d out of range", p->vocab);
    if (p->dim <= 0 || p->dim > kMaxDim || p->dim % 8 != 0)
        return set_error(MORPHO_ERR_INVALID, "cross entropy: dim = %d must be a positive multiple of 8, at most %d", p->dim, kMaxDim);
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

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the backward is cut: columns of a vocabulary piece (a multiple of the tile), and K splits of the
// dhidden (K = piece) and dweight (K = tokens) GEMMs.
struct Cut {
    int cols, pieces, splits_h, splits_w;
};

// K splits of a GEMM of `tiles` tiles and `kb` K blocks in a launch with `total` tile * K-block units on
// `pairs` CTA pairs: no split longer than kMaxK, nor than a third of a pair's share of the launch (so that
// uneven shares cost little), nor, for the latter, shorter than 16 blocks (a partial tile costs about as
// much to write and join as 8 blocks to compute).
int splits_of(int64_t kb, int64_t total, int pairs) {
    const int64_t share = std::max<int64_t>(16, total / (3 * pairs));
    const int64_t splits = ceil_div(kb, std::min<int64_t>(share, kMaxK / BK));
    const int64_t per = ceil_div(kb, splits);
    return static_cast<int>(ceil_div(kb, per));  // no empty split
}

Cut cut_of(const morpho_vocab_loss_t* p, int sms) {
    Cut c;
    const int64_t T = std::max<int64_t>(1, p->tokens);
    const int64_t all = ceil_div(p->vocab, kTile) * kTile;
    const int64_t fit = static_cast<int64_t>(kPieceBytes / 2) / T / kTile * kTile;
    c.cols = static_cast<int>(std::min(all, std::max<int64_t>(kTile, fit)));
    c.pieces = static_cast<int>(ceil_div(p->vocab, c.cols));
    const int64_t tt = ceil_div(T, kTile), tv = c.cols / kTile, td = ceil_div(p->dim, kTile);
    const int64_t total = tt * tv * ceil_div(p->dim, BK) + tt * td * ceil_div(c.cols, BK) + tv * td * ceil_div(T, BK);
    const int pairs = std::max(1, sms / 2);
    c.splits_h = splits_of(ceil_div(std::min<int64_t>(c.cols, p->vocab), BK), total, pairs);
    c.splits_w = splits_of(ceil_div(T, BK), total, pairs);
    return c;
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

// Up to kFewTokens tokens skip the tensor cores; their pieces are the CTAs.
bool few(const morpho_vocab_loss_t* p) {
    return p->tokens <= kFewTokens && p->dim <= kFewMaxDim;
}

int few_blocks(const morpho_vocab_loss_t* p, int sms) { return static_cast<int>(std::min<int64_t>(ceil_div(p->vocab, kFewWarps), sms)); }

int join_rows(int64_t T, int sms) {  // rows a block of the join takes: a power of two up to 32
    int r = 1;
    while (r < 32 && T > static_cast<int64_t>(r) * 2 * sms) r *= 2;
    return r;
}

struct FwdPlan {
    int pieces, rows;
    float2* part;
    float* zt;
    double2* sums;
    uint32_t* done;
};
void plan_forward(Bump& b, const morpho_vocab_loss_t* p, int sms, FwdPlan* f) {
    const size_t T = p->tokens;
    f->pieces = few(p) ? few_blocks(p, sms) : static_cast<int>(ceil_div(p->vocab, kPiece));
    f->rows = join_rows(T, sms);
    f->part = b.take<float2>(f->pieces * T);
    f->zt = b.take<float>(T);
    f->sums = b.take<double2>(ceil_div(T, f->rows));
    f->done = b.take<uint32_t>(1);
}

struct BwdPlan {
    Cut cut;
    uint16_t* dz[2];
    float *common, *hpart, *wpart;
    uint32_t* next;  // a work counter for each launch after the first
    uint8_t* dirty;   // see Clean
    uint16_t* clean;  // (NULL: dhidden, which is written last)
    bool direct;      // dhidden is written by its product, not joined from partial sums
};
void plan_backward(Bump& b, const morpho_vocab_loss_t* p, int sms, BwdPlan* f) {
    f->cut = cut_of(p, sms);
    const Cut& c = f->cut;
    const size_t T = p->tokens, D = p->dim;
    for (int i = 0; i < 2; ++i) f->dz[i] = b.take<uint16_t>(i < c.pieces ? T * c.cols : 0);
    f->common = b.take<float>(1);
    f->next = b.take<uint32_t>(c.pieces);
    f->direct = c.pieces == 1 && c.splits_h == 1;
    f->hpart = b.take<float>(f->direct ? 0 : c.splits_h * T * D);
    f->wpart = b.take<float>(c.splits_w > 1 ? static_cast<size_t>(c.splits_w) * c.cols * D : 0);
    f->dirty = b.take<uint8_t>(ceil_div(T, BK));
    f->clean = f->direct ? b.take<uint16_t>(T * D) : nullptr;
}

int sm_count() {
    DeviceInfo dev;
    const int sms = current_device_info(&dev) == MORPHO_OK ? dev.sms : 148;
    clear_error();
    return sms;
}

// A 16-bit [rows, cols] matrix for loads of 128 x 128 elements as two panels of 64 columns (K-major: 128
// rows, the columns are K; MN-major: 128 of K, the columns are M or N).  Where whole 64-column groups may be
// read (cols a multiple of 64, or rows padded to one) a third dimension over the groups loads both panels
// at once: one thread issues the copies, and with one per panel it was the bottleneck.
int load_map(CUtensorMap* m, bool* whole, const void* base, int64_t rows, int64_t cols, int64_t ld) {
    *whole = cols % 64 == 0;
    if (!*whole) return make_tmap_2d_f16(m, base, rows, cols, ld, 128, 64);
    const uint64_t dims[3] = {64, static_cast<uint64_t>(rows), static_cast<uint64_t>(cols / 64)};
    const uint64_t strides[2] = {static_cast<uint64_t>(ld) * 2, 128};
    const uint32_t box[3] = {64, 128, 2};
    return make_tmap(m, base, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Stores of 32 rows x 64 bytes: a 16-bit matrix, and fp32 slabs [slabs, rows, cols].
int store_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld) {
    return make_tmap_2d_f16(m, base, rows, cols, ld, 32, 32);
}
int slab_map(CUtensorMap* m, const void* base, int64_t slabs, int64_t rows, int64_t cols) {
    const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), static_cast<uint64_t>(slabs)};
    const uint64_t strides[2] = {static_cast<uint64_t>(cols) * 4, static_cast<uint64_t>(rows) * cols * 4};
    const uint32_t box[3] = {16, 32, 1};
    return make_tmap(m, base, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

// Appends a task whose maps are set.
int add_task(Launch* L, Task& t, int kind, bool a_mn, bool b_mn, int64_t M, int64_t N, int64_t K, int splits) {
    t.kind = kind;
    t.a_mn = a_mn;
    t.b_mn = b_mn;
    t.M = static_cast<int>(M);
    t.N = static_cast<int>(N);
    t.tiles_m = static_cast<int>(ceil_div(M, kTile));
    t.tiles_n = static_cast<int>(ceil_div(N, kTile));
    // 16 M tiles x about 5 N tiles at a time on 74 CTA pairs (8 x 9: 2 % slower); a few N tiles run side by side
    t.group = t.tiles_n <= 8 ? 1 : 16;
    t.by_slab = FastDiv::of(t.tiles_m * t.tiles_n);
    t.by_band = FastDiv::of(t.group * t.tiles_n);
    t.by_group = FastDiv::of(t.group);
    t.by_last = FastDiv::of(t.tiles_m % t.group == 0 ? t.group : t.tiles_m % t.group);
    t.K = static_cast<int>(K);
    t.k_blocks = static_cast<int>(ceil_div(K, BK));
    t.kb_per_split = static_cast<int>(ceil_div(t.k_blocks, splits));
    const int64_t before = L->tasks > 0 ? L->task[L->tasks - 1].items_end : 0;
    const int64_t end = before + static_cast<int64_t>(t.tiles_m) * t.tiles_n * ceil_div(t.k_blocks, t.kb_per_split);
    if (end > 2147483647LL - 65536) return set_error(MORPHO_ERR_INVALID, "cross entropy: too many tiles");
    t.items_end = static_cast<int>(end);
    L->task[L->tasks++] = t;
    return MORPHO_OK;
}

// Whether a launch's tiles are taken from a counter as pairs become free, rather than dealt round-robin: an
// item takes 2 us to reach all roles of a pair, which tiles of a few K blocks (0.5 us each) hide and shorter ones do not
// (backward of 3 tokens, 32768 x 1024: 69 us dealt, 72 taken; of 200, 65536 x 2048, 3.6 blocks a tile: 239 and 222).
bool worth_taking(const Launch& L) {
    int64_t units = 0;
    for (int i = 0; i < L.tasks; ++i) units += static_cast<int64_t>(L.task[i].tiles_m) * L.task[i].tiles_n * L.task[i].k_blocks;
    return units >= 3LL * L.task[L.tasks - 1].items_end;
}

template <bool BF16>
int launch(const DeviceInfo& dev, Launch& L, cudaStream_t stream, const char* name) {
    auto kern = vocab_gemm_kernel<BF16>;
    static SharedLimit limit;
    MORPHO_CUDA_TRY(limit.raise(kern, dev.device, kSmemBytes));
    L.status = dev.status;
    const int pairs = std::min(L.task[L.tasks - 1].items_end, std::max(1, dev.sms / 2));
    prof_begin(stream, name);
    MORPHO_CUDA_TRY(launch_after(kern, 2 * pairs, kGemmThreads, kSmemBytes, stream, L));
    MORPHO_LAUNCH_CHECK(name);
    return MORPHO_OK;
}

template <bool BF16>
int finish(const DeviceInfo& dev, const float* part, int slabs, int64_t elems, const float* common, void* out, cudaStream_t stream) {
    prof_begin(stream, "vocab_finish");
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(elems, 2048), 8 * dev.sms));
    MORPHO_CUDA_TRY(launch_after(vocab_finish_kernel<BF16>, grid, 256, 0, stream, part, slabs, elems, common, static_cast<uint16_t*>(out)));
    MORPHO_LAUNCH_CHECK("vocab_finish");
    return MORPHO_OK;
}

template <bool BF16, int TT, int GL, int R>
int launch_few(const DeviceInfo& dev, const Rowwise& r, const morpho_vocab_loss_t* p, const void* hidden, const void* weight, int blocks,
               cudaStream_t stream) {
    static SharedLimit limit;
    const int stage = R * 32 / GL * 2 * p->dim;
    const int stages = std::max(1, std::min(kFewMaxStages, kFewRing / (kFewWarps * stage)));
    const int smem = kFewWarps * stages * stage + TT * 2 * p->dim;
    auto kern = vocab_few_kernel<BF16, TT, GL, R>;
    MORPHO_CUDA_TRY(limit.raise(kern, dev.device, smem));
    prof_begin(stream, "vocab_few");
    MORPHO_CUDA_TRY(launch_after(kern, blocks, kFewThreads, smem, stream, r, static_cast<const uint16_t*>(hidden), ld_hidden(p),
                                 static_cast<const uint16_t*>(weight), ld_weight(p), p->dim, stages, dev.status));
    MORPHO_LAUNCH_CHECK("vocab_few");
    return MORPHO_OK;
}

// Lanes to a row: so many rows at a time that every warp has three stages of them in the ring.
template <bool BF16, int TT>
int launch_few(const DeviceInfo& dev, const Rowwise& r, const morpho_vocab_loss_t* p, const void* hidden, const void* weight, int blocks,
               cudaStream_t stream) {
    return p->dim <= 512    ? launch_few<BF16, TT, 8, 2>(dev, r, p, hidden, weight, blocks, stream)
           : p->dim <= 1024 ? launch_few<BF16, TT, 8, 1>(dev, r, p, hidden, weight, blocks, stream)
           : p->dim <= 2048 ? launch_few<BF16, TT, 16, 1>(dev, r, p, hidden, weight, blocks, stream)
                            : launch_few<BF16, TT, 32, 1>(dev, r, p, hidden, weight, blocks, stream);
}

int launch_join(const Rowwise& r, const FwdPlan& f, float* loss, float* lse, cudaStream_t stream) {
    prof_begin(stream, "vocab_join");
    const unsigned grid = static_cast<unsigned>(ceil_div(r.T, f.rows));
    auto go = [&](auto kern) { return launch_after(kern, grid, kJoinThreads, 0, stream, r, f.pieces, f.sums, loss, lse); };
    MORPHO_CUDA_TRY(f.rows == 1    ? go(vocab_join_kernel<1>)
                    : f.rows == 2  ? go(vocab_join_kernel<2>)
                    : f.rows == 4  ? go(vocab_join_kernel<4>)
                    : f.rows == 8  ? go(vocab_join_kernel<8>)
                    : f.rows == 16 ? go(vocab_join_kernel<16>)
                                   : go(vocab_join_kernel<32>));
    MORPHO_LAUNCH_CHECK("vocab_join");
    return MORPHO_OK;
}

// The tensor core truncates its fp32 accumulator after every K = 16 step: on average half a unit in the last
// place of the running sum is lost, always towards zero.  For a sum that grows evenly to z in n steps these
// units average 0.35 2^-23 z, so z comes out short by n 2.1e-8 of itself (measured 1.5e-8 in bf16, where
// early sums are exact, and 1.9e-8 in fp16); 1.8e-8 is put back.  At dim 1024 that takes the error of a
// target's logit from 8e-6 to that of an fp32 sum, 3e-6.  The constant is fitted to sums whose terms are alike.  Where
// nothing is truncated (a hidden row with a few non-zero elements) it is itself the error: 1.2e-6 of the logit
// at dim 1024, 1.8e-5 at 16384, which is what the other sums would be short by without it.
float unbias_of(int dim) { return static_cast<float>(1.0 + (dim + 15) / 16 * 1.8e-8); }

Rowwise rows_of(const morpho_vocab_loss_t* p, const int64_t* target) {
    Rowwise r{};
    r.unbias = unbias_of(p->dim);
    r.log2e = static_cast<float>(1.4426950408889634 * (1.0 + (p->dim + 15) / 16 * 1.8e-8));
    r.T = p->tokens;
    r.V = p->vocab;
    r.target = target;
    r.ignore_index = p->ignore_index;
    r.reduction = p->reduction;
    return r;
}

template <bool BF16>
int forward_t(const DeviceInfo& dev, const morpho_vocab_loss_t* p, const void* hidden, const void* weight, const int64_t* target,
              float* loss, float* lse, const FwdPlan& f, cudaStream_t stream) {
    Rowwise r = rows_of(p, target);
    r.part = f.part;
    r.zt = f.zt;
    r.done = f.done;
    if (few(p)) {
        MORPHO_TRY(p->tokens == 1 ? (launch_few<BF16, 1>(dev, r, p, hidden, weight, f.pieces, stream))
                                  : (launch_few<BF16, 2>(dev, r, p, hidden, weight, f.pieces, stream)));
    } else {
        Launch L{};
        L.rows = r;
        Task t{};
        MORPHO_TRY(load_map(&t.a, &t.a_whole, hidden, p->tokens, p->dim, ld_hidden(p)));
        MORPHO_TRY(load_map(&t.b, &t.b_whole, weight, p->vocab, p->dim, ld_weight(p)));
        MORPHO_TRY(add_task(&L, t, kStats, false, false, p->tokens, p->vocab, p->dim, 1));
        MORPHO_TRY(launch<BF16>(dev, L, stream, "vocab_stats"));
    }
    return launch_join(r, f, loss, lse, stream);
}

// One launch computes dz of piece i + 1 beside the two products that read dz of piece i (the two dz
// buffers alternate), so the tiles of all three fill the SMs together.
template <bool BF16>
int backward_t(const DeviceInfo& dev, const morpho_vocab_loss_t* p, const float* grad, const void* hidden, const void* weight,
               const int64_t* target, const float* lse, void* dhidden, void* dweight, const BwdPlan& f, cudaStream_t stream) {
    Rowwise r = rows_of(p, target);
    r.lse = lse;
    r.grad = grad;
    r.unit = BF16 ? 1.0f : 32768.0f;
    r.log2_unit = BF16 ? 0.0f : 15.0f;
    r.common = f.common;
    const Cut& c = f.cut;
    const int64_t T = p->tokens, D = p->dim;
    uint16_t* clean = f.clean != nullptr ? f.clean : static_cast<uint16_t*>(dhidden);
    auto width = [&](int i) { return std::min<int64_t>(c.cols, p->vocab - static_cast<int64_t>(i) * c.cols); };
    for (int i = -1; i < c.pieces; ++i) {
        Launch L{};
        L.rows = r;
        bool mixed = false;  // tiles of different lengths
        L.rows.first = i < 0;
        if (i >= 0) {
            const int v0 = i * c.cols;
            const int64_t n = width(i), padded = ceil_div(n, 64) * 64;  // dz holds zeros up to whole panels
            Task w{}, h{};
            uint16_t* dw = static_cast<uint16_t*>(dweight) + static_cast<int64_t>(v0) * D;
            MORPHO_TRY(load_map(&w.a, &w.a_whole, f.dz[i & 1], T, padded, c.cols));
            MORPHO_TRY(load_map(&w.b, &w.b_whole, hidden, T, D, ld_hidden(p)));
            if (c.splits_w > 1)
                MORPHO_TRY(slab_map(&w.out, f.wpart, c.splits_w, n, D));
            else
                MORPHO_TRY(store_map(&w.out, dw, n, D, D));
            MORPHO_TRY(load_map(&h.a, &h.a_whole, f.dz[i & 1], T, padded, c.cols));
            MORPHO_TRY(load_map(&h.b, &h.b_whole, weight, p->vocab, D, ld_weight(p)));
            h.b_row0 = v0;
            w.dirty = f.dirty;
            MORPHO_TRY(load_map(&L.clean, &w.b_whole, clean, T, D, D));
            if (f.direct)
                MORPHO_TRY(store_map(&h.out, dhidden, T, D, D));
            else
                MORPHO_TRY(slab_map(&h.out, f.hpart, c.splits_h, T, D));
            // a shorter last piece may have fewer splits: the other slabs keep the earlier pieces' sums
            const int splits_h = static_cast<int>(std::min<int64_t>(c.splits_h, ceil_div(n, BK)));
            auto add_w = [&]() { return add_task(&L, w, c.splits_w > 1 ? kPart : kOut, true, true, n, D, T, c.splits_w); };
            auto add_h = [&]() { return add_task(&L, h, f.direct ? kOut : i == 0 ? kPart : kPartAdd, false, true, T, D, n, splits_h); };
            // the longest items first: the pairs that finish early take the short ones (dz last)
            const bool h_first = ceil_div(n, splits_h) > ceil_div(T, c.splits_w);
            MORPHO_TRY(h_first ? add_h() : add_w());
            MORPHO_TRY(h_first ? add_w() : add_h());
            mixed = true;
        } else {
            L.zero = f.next;
            L.zeros = c.pieces;
            L.cleaning = Clean{static_cast<const uint16_t*>(hidden), ld_hidden(p), static_cast<int>(D), static_cast<int>(ceil_div(T, BK)), clean, f.dirty};
        }
        if (i + 1 < c.pieces) {
            Task z{};
            z.v0 = (i + 1) * c.cols;
            z.b_row0 = z.v0;
            z.padded = static_cast<int>(ceil_div(width(i + 1), 64) * 64);
            MORPHO_TRY(load_map(&z.a, &z.a_whole, hidden, T, D, ld_hidden(p)));
            MORPHO_TRY(load_map(&z.b, &z.b_whole, weight, p->vocab, D, ld_weight(p)));
            MORPHO_TRY(store_map(&z.out, f.dz[(i + 1) & 1], T, z.padded, c.cols));
            MORPHO_TRY(add_task(&L, z, kDz, false, false, T, width(i + 1), D, 1));
        }
        if (mixed && worth_taking(L)) L.next = f.next + i;
        MORPHO_TRY(launch<BF16>(dev, L, stream, i < 0 ? "vocab_dz" : "vocab_grad"));
        if (i >= 0 && c.splits_w > 1)
            MORPHO_TRY(finish<BF16>(dev, f.wpart, c.splits_w, width(i) * D, f.common,
                                    static_cast<uint16_t*>(dweight) + static_cast<int64_t>(i) * c.cols * D, stream));
    }
    if (!f.direct) MORPHO_TRY(finish<BF16>(dev, f.hpart, c.splits_h, T * D, f.common, dhidden, stream));
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
    plan_forward(b, p, sm_count(), &f);
    return b.off + 256;
}

extern "C" MORPHO_API size_t morpho_sm100_linear_cross_entropy_backward_workspace_size(const morpho_vocab_loss_t* p) {
    clear_error();
    if (validate_loss(p) != MORPHO_OK) return 0;
    Bump b{nullptr};
    BwdPlan f;
    plan_backward(b, p, sm_count(), &f);
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
    plan_forward(b, p, dev.sms, &f);
    return p->type == MORPHO_DTYPE_BF16 ? forward_t<true>(dev, p, hidden, weight, target, loss, lse, f, st)
                                        : forward_t<false>(dev, p, hidden, weight, target, loss, lse, f, st);
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
    plan_backward(b, p, dev.sms, &f);
    return p->type == MORPHO_DTYPE_BF16 ? backward_t<true>(dev, p, grad_loss, hidden, weight, target, lse, dhidden, dweight, f, st)
                                        : backward_t<false>(dev, p, grad_loss, hidden, weight, target, lse, dhidden, dweight, f, st);
}
