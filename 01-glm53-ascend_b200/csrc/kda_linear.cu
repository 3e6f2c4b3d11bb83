// The attention layer's projections on sm_100a, behind kda_linear_launch:
//   out[t, n] = round(act(sx[t] sw[n] sum_k x[t, k] w[n, k] + bias[n]) + residual[t, n])
// bf16, fp16 or e4m3 operands, fp32 sums in tensor memory. Both operands are
// K-contiguous, so every operand tile is rows of 128 bytes along K, brought in
// by tiled TMA with the 128-byte swizzle; in bytes the three types are alike,
// and only the tcgen05 kind and its descriptor differ.
//
// Two kernels:
//   * pair_kernel, for many tokens: persistent pairs of CTAs (cta_group::2),
//     256 tokens x 64..256 outputs per tile, tokens on the tensor memory's
//     lanes. Bound by the tensor cores (2 T K N operations) for long K, by the
//     output's bytes for short K. A tile of 256 x 256 brings 32 KB to each SM per
//     128-byte block of K and its 512 cycles of products; two accumulators let the
//     next tile's products run under the epilogue. 8256 x 12576 x 4096 bf16:
//     1,300 TFLOP/s at the power limit (the tensor pipe 90 to 92% active on 4096 x
//     9216); 33494 x 4096 x 4096 e4m3 with residual: 2,300 TFLOP/s.
//   * narrow_kernel, for few tokens, where the weights' bytes are the work:
//     128 outputs on the lanes x 16..64 tokens as the columns, so that a tile of
//     weights is read once; K split over the CTAs of a cluster, which keeps every
//     SM reading, and joined through distributed shared memory in a fixed order, so
//     results repeat bit for bit. 64 x 12576 x 4096 bf16 with weights that no
//     earlier launch left in L2: 22.9 us, 4.5 TB/s; 1 x 4096 x 4096 e4m3: 6.2 us, of
//     which the weights' bytes are 2.6 at HBM's rate, the rest first load, join and launch.
// Operands whose rows do not start on 16-byte boundaries, which TMA needs, are
// first copied to rows that do (realign_kernel).

#include <cuda.h>

#include <climits>

#include "kda_host.cuh"
#include "kda_rows.cuh"

namespace kda {
namespace linear {

// ---------------------------------------------------------------------------
// PTX: clusters, tiled TMA, tcgen05
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// True in one lane of the (converged) warp. Code under it is known to run in a
// single thread, so the tensor-core and TMA instructions, which take uniform
// registers, issue without a loop over the lanes (600 -> 340 cycles for a stage
// of four products and its commit).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The two halves of a barrier that orders no memory.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// The address in CTA `rank` of the cluster that corresponds to `addr` here.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 load_peer(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void store_peer(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// An arrival on a barrier of the pair. It hands over tensor memory that has been
// read, no ordinary memory, so it need not wait for this thread's stores as a
// release over the cluster does (1 us here).
__device__ __forceinline__ void arrive_peer(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// 2-D tiled loads (x = K column, y = row) and stores. No TMA multicast.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// The same into this CTA's memory, counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// The box on its way into L2 only. L2 is where global memory is coherent, so this
// may run ahead of the kernels before: what they still write is not missed.
__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap *map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// This thread's committed stores have read shared memory.
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t columns) {
    if constexpr (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D[tmem] (+)= A[smem] B[smem]; E4M3 picks the kind, CTAS the CTAs of one product.
template <int CTAS, bool E4M3>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define KDA_MMA(group, kind)                                                                            \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma." group "." kind           \
                 " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)     \
                 : "memory")
    if constexpr (CTAS == 2 && E4M3) KDA_MMA("cta_group::2", "kind::f8f6f4");
    if constexpr (CTAS == 2 && !E4M3) KDA_MMA("cta_group::2", "kind::f16");
    if constexpr (CTAS == 1 && E4M3) KDA_MMA("cta_group::1", "kind::f8f6f4");
    if constexpr (CTAS == 1 && !E4M3) KDA_MMA("cta_group::1", "kind::f16");
#undef KDA_MMA
}
// This thread's products so far arrive on `bar` when complete: here, or in both CTAs of the pair.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_commit_pair(uint32_t bar, uint16_t ctas) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(ctas)
        : "memory");
}

// 32 consecutive fp32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory descriptor of a K-major tile of 128-byte rows in the 128-byte
// swizzle (8-row groups 1024 bytes apart). 32 bytes of K further along is + 2.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: fp32 sums, both operands of one type (`format`: 1 for
// bf16; 0 for fp16, and for e4m3 in its kind).
__host__ __device__ constexpr uint32_t instruction_desc(int m, int n, uint32_t format) {
    return (1u << 4) | (format << 7) | (format << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// ---------------------------------------------------------------------------
// Epilogue arithmetic
// ---------------------------------------------------------------------------

template <int ACT, int N>
__device__ __forceinline__ void activate_all(float2 (&y)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = activate2<ACT>(y[i]);
}
template <int N>
__device__ __forceinline__ void activate_all(int act, float2 (&y)[N]) {
    switch (act) {
        case KDA_ACT_SILU: activate_all<KDA_ACT_SILU>(y); break;
        case KDA_ACT_SIGMOID: activate_all<KDA_ACT_SIGMOID>(y); break;
        case KDA_ACT_RELU: activate_all<KDA_ACT_RELU>(y); break;
        case KDA_ACT_GELU_TANH: activate_all<KDA_ACT_GELU_TANH>(y); break;
        default: break;
    }
}
// v[n .. n + 3] of an fp32 vector of `size` values (zeros past the end), alike in every lane.
__device__ __forceinline__ float4 vector4(const float *v, int64_t n, int64_t size, bool aligned) {
    if (aligned && n + 4 <= size) return *reinterpret_cast<const float4 *>(v + n);
    return make_float4(n < size ? v[n] : 0.0f, n + 1 < size ? v[n + 1] : 0.0f, n + 2 < size ? v[n + 2] : 0.0f,
                       n + 3 < size ? v[n + 3] : 0.0f);
}

// mbar_wait without its suspension, for the two threads that keep the tensor
// cores fed: a wake-up costs more than a poll where a stage is short (4096 x
// 9216 x 4096 bf16 at width 128: 250 us against 275; at 256 both 203). Bounded alike.
__device__ __forceinline__ bool mbar_spin(uint64_t *bar, uint32_t phase, int32_t *status, volatile int32_t *abort) {
    const uint32_t addr = smem_addr(bar);
    for (uint32_t i = 0; i < 1u << 27; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(addr), "r"(phase)
            : "memory");
        if (done != 0) return true;
        if ((i & 255) == 255 && *abort != 0) return false;
    }
    *abort = 1;
    report(status, KDA_DEVICE_ERR_WAIT_TIMEOUT);
    return false;
}

// What one launch needs besides its arguments.
struct Maps {
    CUtensorMap x, weight, out, residual;
};
struct Plan {
    int32_t k_blocks;        // 128-byte blocks of K
    int32_t tiles_t, tiles_n;
    uint32_t idesc, idesc_tail;      // of a whole tile, and of the last one along N (pair_kernel)
    int32_t width, tail;             // their columns: width a multiple of 64, tail of 32
    int32_t out_tma, residual_tma;   // rows that TMA can store and load (narrow_kernel: that start on 16 bytes)
    int32_t vectors;                 // bias and weight scale start on 16 bytes
};

constexpr int kRowBytes = 128;       // bytes of K per block and operand row
constexpr int kLanes = 128;          // tensor-memory lanes

// ---------------------------------------------------------------------------
// pair_kernel
// ---------------------------------------------------------------------------

struct Pair {
    static constexpr int kTileT = 256;                        // tokens per tile, 128 per CTA
    static constexpr int kMaxN = 256;                         // outputs per tile at most
    static constexpr int kBytesX = kLanes * kRowBytes;        // per CTA and stage
    static constexpr int kBytesW = kMaxN / 2 * kRowBytes;     // half of the weights' rows
    static constexpr int kStageBytes = kBytesX + kBytesW;
    static constexpr int kStages = 5;
    static constexpr int kBoxBytes = 32 * 128;                // 64 outputs of a warp's 32 tokens
    static constexpr int kEpilogueWarps = 16;                 // 4 of 32 tokens x 4 boxes of 64 outputs
    static constexpr int kThreads = 32 * (kEpilogueWarps + 2);
    static constexpr int kColumns = 2 * kMaxN;                // two accumulators
    static constexpr int kStaging = kStages * kStageBytes;    // a box per epilogue warp
    static constexpr int kVectors = kStaging + kEpilogueWarps * kBoxBytes;   // bias or weight scale, 32 columns a warp
    static constexpr int kBars = kVectors + kEpilogueWarps * 32 * 4;
    static constexpr int kNumBars = 2 * kStages + 4 + kEpilogueWarps + 1;
    static constexpr int kBytes = kBars + kNumBars * 8 + 16;
    static_assert(kBytes <= 227 * 1024, "one CTA's shared memory");
};

// Tile `i` in an order that keeps the operands of the tiles in flight few:
// strips of 8 token tiles, the token tile running fastest. 33494 x 12576 x 4096
// e4m3: 1,415 us in strips of 1, 2 or 4, 1,367 of 8, 1,362 of 16, 1,372 of 32; 33494 x
// 4096 x 4096 436 up to 8, 441 beyond.
__device__ __forceinline__ void tile_at(int i, int tiles_t, int tiles_n, int &t, int &n) {
    constexpr int kStrip = 8;
    const int strip = i / (kStrip * tiles_n), first = strip * kStrip;
    const int height = min(kStrip, tiles_t - first), in = i - first * tiles_n;
    t = first + in % height;
    n = in / height;
}

// A warp's box of up to 32 rows x 64 columns in the 128-byte swizzle, from and to
// rows off 16-byte boundaries: elements side by side along a row, 16 accesses
// of a lane in flight.
template <typename O>
__device__ __forceinline__ O *box_at(uint8_t *box, int r, int j) {
    return reinterpret_cast<O *>(box + r * 128 + (((j >> 3) ^ (r & 7)) << 4) + (j & 7) * 2);
}
template <typename O>
__device__ __forceinline__ void rows_to_box(const O *src, int64_t stride, uint8_t *box, int64_t rows, int64_t columns) {
    const int lane = threadIdx.x & 31;
    for (int r0 = 0; r0 < 32; r0 += 8) {
        O v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = r0 + i / 2, j = i % 2 * 32 + lane;
            if (r < rows && j < columns) v[i] = src[r * stride + j];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) *box_at<O>(box, r0 + i / 2, i % 2 * 32 + lane) = v[i];
    }
}
template <typename O>
__device__ __forceinline__ void box_to_rows(uint8_t *box, O *dst, int64_t stride, int64_t rows, int64_t columns) {
    const int lane = threadIdx.x & 31;
    for (int r0 = 0; r0 < 32; r0 += 8) {
        O v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = *box_at<O>(box, r0 + i / 2, i % 2 * 32 + lane);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = r0 + i / 2, j = i % 2 * 32 + lane;
            if (r < rows && j < columns) dst[r * stride + j] = v[i];
        }
    }
}

// TMA_ROWS: out, and residual where there is one, are rows that TMA stores and
// loads (a store's width a multiple of 16 bytes). The general form holds more registers (3-5% on large products).
template <typename O, bool E4M3, bool TMA_ROWS>
__global__ void __launch_bounds__(Pair::kThreads, 1)
    pair_kernel(const KdaLinearArgs p, const Plan plan, const __grid_constant__ Maps maps) {
    using C = Pair;
    extern __shared__ __align__(1024) uint8_t smem[];   // the swizzle's atom
    const uint32_t base = smem_addr(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBars);
    uint64_t *full = bars, *empty = bars + C::kStages, *tfull = bars + 2 * C::kStages, *tempty = tfull + 2;
    uint64_t *rfull = tempty + 2, *drain = rfull + C::kEpilogueWarps;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::kNumBars);
    volatile int32_t *abort_word = reinterpret_cast<volatile int32_t *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();

    let_next_start();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 2 * C::kEpilogueWarps);
        }
        for (int i = 0; i < C::kEpilogueWarps; ++i) mbar_init(&rfull[i], 1);
        mbar_init(drain, 1);
        *abort_word = 0;
        fence_mbar_init();
        prefetch_map(&maps.x);
        prefetch_map(&maps.weight);
    }
    constexpr int kBlock = E4M3 ? kRowBytes : kRowBytes / 2;   // elements of K
    const int tiles = plan.tiles_t * plan.tiles_n, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    if (warp == C::kEpilogueWarps + 1) tmem_alloc<2>(tmem_slot, C::kColumns);
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    wait_for_previous();
    const uint32_t tmem = *tmem_slot;

    if (warp == C::kEpilogueWarps) {
        // Loads: this CTA's 128 token rows and its half of the weight rows, counted in the first CTA.
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = first; i < tiles && ok; i += step) {
                int t, n;
                tile_at(i, plan.tiles_t, plan.tiles_n, t, n);
                const int row_x = t * C::kTileT + rank * kLanes, row_w = n * plan.width + rank * ((n + 1 == plan.tiles_n ? plan.tail : plan.width) / 2);
                for (int kb = 0; kb < plan.k_blocks; ++kb) {
                    if (!mbar_spin(&empty[stage], phase ^ 1, p.status, abort_word)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = peer_addr(smem_addr(&full[stage]), 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * (C::kBytesX + plan.width / 2 * kRowBytes));
                    const uint32_t dst = base + stage * C::kStageBytes;
                    const int k = kb * kBlock;
                    tma_load_pair(dst, &maps.x, k, row_x, bar);
                    tma_load_pair(dst + C::kBytesX, &maps.weight, k, row_w, bar);
                    if (++stage == C::kStages) stage = 0, phase ^= 1;
                }
            }
            // Every stage is free again (its copies landed and were read) before this CTA may go. After an
            // expired wait one full wait gives the copies in flight the time to land.
            if (!ok) mbar_wait(&empty[stage], phase ^ 1, p.status);
            for (int i = 0; i < C::kStages && ok; ++i) {
                ok = mbar_wait(&empty[stage], phase ^ 1, p.status, abort_word);
                if (++stage == C::kStages) stage = 0, phase ^= 1;
            }
        }
    } else if (warp == C::kEpilogueWarps + 1) {
        // Products: one thread of the first CTA for both.
        if (rank == 0 && elect_one()) {
            int stage = 0, buffer = 0;
            uint32_t phase = 0, tphase = 0;
            bool ok = true;
            for (int i = first; i < tiles && ok; i += step) {
                ok = mbar_wait(&tempty[buffer], tphase ^ 1, p.status, abort_word);
                if (!ok) break;
                tc_fence_after();
                int t, n;
                tile_at(i, plan.tiles_t, plan.tiles_n, t, n);
                const uint32_t d = tmem + buffer * C::kMaxN, idesc = n + 1 == plan.tiles_n ? plan.idesc_tail : plan.idesc;
                for (int kb = 0; kb < plan.k_blocks; ++kb) {
                    ok = mbar_spin(&full[stage], phase, p.status, abort_word);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t a = operand_desc(base + stage * C::kStageBytes);
                    const uint64_t b = operand_desc(base + stage * C::kStageBytes + C::kBytesX);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma<2, E4M3>(d, a + 2 * k, b + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
                    mma_commit_pair(smem_addr(&empty[stage]), 3);
                    if (++stage == C::kStages) stage = 0, phase ^= 1;
                }
                mma_commit_pair(smem_addr(&tfull[buffer]), 3);
                if (++buffer == 2) buffer = 0, tphase ^= 1;
            }
            mma_commit_pair(smem_addr(drain), 1);
            mbar_wait(drain, 0, p.status);
        }
    } else {
        // Epilogue: a warp has 32 tokens (its quarter of the lanes) and one box of 64 columns, staged in its own
        // shared memory, so that no warp waits for another. 16 warps, as each has long chains of dependent
        // instructions: with 8 of two boxes each, 8256 x 4096 outputs of K = 128 took 21.0 us instead of 17.5.
        const int quarter = warp & 3, group = warp >> 2;
        uint8_t *stage = smem + C::kStaging + warp * C::kBoxBytes;
        const uint32_t stage_addr = base + C::kStaging + warp * C::kBoxBytes;
        float *vector = reinterpret_cast<float *>(smem + C::kVectors) + warp * 32;
        const O *residual = static_cast<const O *>(p.residual);
        O *out = static_cast<O *>(p.out);
        const bool residual_tma = TMA_ROWS ? residual != nullptr : plan.residual_tma != 0;
        const bool has_box = group * 64 < plan.width;
        int buffer = 0;
        uint32_t tphase = 0, rphase = 0;
        for (int i = first; i < tiles; i += step) {
            int t, n;
            tile_at(i, plan.tiles_t, plan.tiles_n, t, n);
            const int64_t t0 = static_cast<int64_t>(t) * C::kTileT + rank * kLanes + quarter * 32;
            const int64_t n0 = static_cast<int64_t>(n) * plan.width + group * 64;
            const bool any = has_box && t0 < p.num_tokens && n0 < p.out_features;
            if (residual_tma && any && lane == 0) {
                bulk_wait_read();   // the last tile's store has left the box
                mbar_arrive_expect_tx(&rfull[warp], C::kBoxBytes);
                tma_load(stage_addr, &maps.residual, static_cast<int>(n0), static_cast<int>(t0), smem_addr(&rfull[warp]));
            }
            if (!TMA_ROWS && residual != nullptr && !residual_tma && any) {
                if (lane == 0) bulk_wait_read();
                __syncwarp();
                rows_to_box<O>(residual + t0 * p.residual_row_stride + n0, p.residual_row_stride, stage, p.num_tokens - t0,
                               p.out_features - n0);
                __syncwarp();
            }
            // This lane's row scale, and of each 32 columns one column's bias and scale, on their way while the products run.
            const float sx = E4M3 && t0 + lane < p.num_tokens ? p.x_scale[t0 + lane] : 0.0f;
            float bias[2], scale[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t at = n0 + h * 32 + lane;
                bias[h] = any && p.bias != nullptr && at < p.out_features ? p.bias[at] : 0.0f;
                scale[h] = E4M3 && any && at < p.out_features ? p.weight_scale[at] : 0.0f;
            }
            bool ok = mbar_wait(&tfull[buffer], tphase, p.status, abort_word);
            if (residual_tma && any) {
                // Waited for even after an expired wait: the copy must land before the CTA may go.
                ok = mbar_wait(&rfull[warp], rphase, p.status) && ok;
                rphase ^= 1;
            }
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint32_t columns = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buffer * C::kMaxN + group * 64;
            const uint32_t done = peer_addr(smem_addr(&tempty[buffer]), 0);
            if (++buffer == 2) buffer = 0, tphase ^= 1;
            if (!any) {
                if (lane == 0) arrive_peer(done);
                continue;
            }
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                uint32_t acc[32];
                tmem_load32(columns + h * 32, acc);
                tmem_wait_load();
                if (h == 1) {
                    // The accumulator is in registers: the next tile's products may start.
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_peer(done);
                }
                float2 y[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = make_float2(__uint_as_float(acc[2 * j]), __uint_as_float(acc[2 * j + 1]));
                if (E4M3) {
                    // The weight's scale, then the token's: their product alone may pass fp32's range. The token's by
                    // single values, as pairs of it cost registers (8256 x 4096 outputs of K = 128: 19.6 us; by pairs,
                    // spilled, 31).
                    const auto scaled = [&](float2 v) { return make_float2(v.x * sx, v.y * sx); };
                    vector[lane] = h == 0 ? scale[0] : scale[1];
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 s = *reinterpret_cast<const float4 *>(vector + 4 * j);
                        y[2 * j] = scaled(mul2(y[2 * j], make_float2(s.x, s.y)));
                        y[2 * j + 1] = scaled(mul2(y[2 * j + 1], make_float2(s.z, s.w)));
                    }
                    __syncwarp();
                }
                if (p.bias != nullptr) {
                    vector[lane] = h == 0 ? bias[0] : bias[1];
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 b = *reinterpret_cast<const float4 *>(vector + 4 * j);
                        y[2 * j] = add2(y[2 * j], make_float2(b.x, b.y));
                        y[2 * j + 1] = add2(y[2 * j + 1], make_float2(b.z, b.w));
                    }
                    __syncwarp();
                }
                activate_all(p.activation, y);
                if (h == 0 && residual == nullptr) {
                    if (lane == 0) bulk_wait_read();   // as late as it can be
                    __syncwarp();
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    uint4 *at = reinterpret_cast<uint4 *>(stage + lane * 128 + (((h * 4 + v) ^ (lane & 7)) << 4));
                    if (residual != nullptr) {
                        const uint4 r = *at;
                        y[v * 4] = add2(y[v * 4], unpack2<O>(r.x));
                        y[v * 4 + 1] = add2(y[v * 4 + 1], unpack2<O>(r.y));
                        y[v * 4 + 2] = add2(y[v * 4 + 2], unpack2<O>(r.z));
                        y[v * 4 + 3] = add2(y[v * 4 + 3], unpack2<O>(r.w));
                    }
                    *at = make_uint4(pack2<O>(y[v * 4].x, y[v * 4].y), pack2<O>(y[v * 4 + 1].x, y[v * 4 + 1].y),
                                     pack2<O>(y[v * 4 + 2].x, y[v * 4 + 2].y), pack2<O>(y[v * 4 + 3].x, y[v * 4 + 3].y));
                }
            }
            fence_async_smem();   // the box goes to the store, or to the next residual copy
            __syncwarp();
            if (TMA_ROWS || plan.out_tma) {
                if (lane == 0) {
                    tma_store(&maps.out, stage_addr, static_cast<int>(n0), static_cast<int>(t0));
                    bulk_commit();
                }
            } else {
                box_to_rows<O>(stage, out + t0 * p.out_row_stride + n0, p.out_row_stride, p.num_tokens - t0,
                               p.out_features - n0);
                fence_async_smem();
                __syncwarp();
            }
        }
        if (lane == 0) bulk_wait();
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    if (warp == C::kEpilogueWarps + 1) tmem_free<2>(tmem, C::kColumns);
}

// ---------------------------------------------------------------------------
// narrow_kernel
// ---------------------------------------------------------------------------

// Blocks of K of the weights that a CTA asks into L2 before it waits for the
// kernel before it: with 4, one token through 4096 x 4096 bf16 took 9.2 us instead
// of 9.9; 16 cost 64 tokens through 12576 x 4096 1 us.
constexpr int kAhead = 4;

// How the splits' sums meet. SEND: each CTA stores its sums into the memory of
// the CTA that joins the token, which costs operand stages for an inbox but only one
// barrier. Otherwise a CTA's sums stay where its stages were and the joining
// CTA loads them, with a barrier on both sides. Sending pays where each CTA
// joins 8 tokens at most, which the rule below gives with 16 tokens a tile only
// (bf16, K = 4096, N = 4096, tile/splits: 1 token, 16/4 8.2 us against 9.3; 64
// tokens, 16/2 13.0 against 13.5; 128 tokens, 32/2 15.6 against 14.4).
template <int BT, bool SEND>
struct Narrow {
    static constexpr int kBytesW = kLanes * kRowBytes;
    static constexpr int kBytesX = BT * kRowBytes;
    static constexpr int kStageBytes = kBytesW + kBytesX;
    static constexpr int kStages = BT <= 16 ? (SEND ? 5 : 6) : BT <= 32 ? 5 : 4;
    static constexpr int kThreads = 32 * 6;                   // 4 epilogue warps, loads, products
    static constexpr int kColumns = BT < 32 ? 32 : BT;
    static constexpr int kMaxSplits = 8;
    // The sums: the inbox (tokens x splits rows of 128, each CTA's tokens rounded up), or the stages again.
    static constexpr int kSums = SEND ? kStages * kStageBytes : 0;
    static constexpr int kSumsEnd = kSums + (SEND ? BT + kMaxSplits - 1 : BT) * kLanes * 4;
    static constexpr int kScales = kSumsEnd > kStages * kStageBytes ? kSumsEnd : kStages * kStageBytes;   // the tokens' scales
    static constexpr int kBars = kScales + BT * 4;
    static constexpr int kNumBars = 2 * kStages + 1;
    static constexpr int kBytes = kBars + kNumBars * 8 + 16;
    static_assert(2 * (kBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};

template <typename O, bool E4M3, int BT, bool SEND>
__global__ void __launch_bounds__(Narrow<BT, SEND>::kThreads)
    narrow_kernel(const KdaLinearArgs p, const Plan plan, const int splits, const __grid_constant__ Maps maps) {
    using C = Narrow<BT, SEND>;
    extern __shared__ __align__(1024) uint8_t smem[];   // the swizzle's atom
    const uint32_t base = smem_addr(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBars);
    uint64_t *full = bars, *empty = bars + C::kStages, *tfull = bars + 2 * C::kStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::kNumBars);
    volatile int32_t *abort_word = reinterpret_cast<volatile int32_t *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % splits, tile_n = blockIdx.x / splits;   // split = rank in the cluster
    const int64_t n0 = static_cast<int64_t>(tile_n) * kLanes, t0 = static_cast<int64_t>(blockIdx.y) * BT;
    const int first = static_cast<int>(static_cast<int64_t>(plan.k_blocks) * split / splits);
    const int last = static_cast<int>(static_cast<int64_t>(plan.k_blocks) * (split + 1) / splits);   // > first

    let_next_start();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(tfull, 1);
        *abort_word = 0;
        fence_mbar_init();
        prefetch_map(&maps.x);
        prefetch_map(&maps.weight);
    }
    constexpr int kBlock = E4M3 ? kRowBytes : kRowBytes / 2;   // elements of K
    if (warp == 4 && elect_one())
        for (int kb = first; kb < last && kb < first + kAhead; ++kb) tma_prefetch(&maps.weight, kb * kBlock, static_cast<int>(n0));
    if (warp == 5) tmem_alloc<1>(tmem_slot, C::kColumns);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (SEND) cluster_arrive();
    wait_for_previous();
    const uint32_t tmem = *tmem_slot;

    if (warp == 4) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = first; kb < last; ++kb) {
                if (!mbar_spin(&empty[stage], phase ^ 1, p.status, abort_word)) {
                    // Copies in flight: one full wait gives them the time to land.
                    mbar_wait(&empty[stage], phase ^ 1, p.status);
                    break;
                }
                mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
                const uint32_t dst = base + stage * C::kStageBytes, bar = smem_addr(&full[stage]);
                const int k = kb * kBlock;
                tma_load(dst, &maps.weight, k, static_cast<int>(n0), bar);
                tma_load(dst + C::kBytesW, &maps.x, k, static_cast<int>(t0), bar);
                if (++stage == C::kStages) stage = 0, phase ^= 1;
            }
        }
    } else if (warp == 5) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = first; kb < last; ++kb) {
                if (!mbar_spin(&full[stage], phase, p.status, abort_word)) break;
                tc_fence_after();
                const uint64_t a = operand_desc(base + stage * C::kStageBytes);
                const uint64_t b = operand_desc(base + stage * C::kStageBytes + C::kBytesW);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma<1, E4M3>(tmem, a + 2 * k, b + 2 * k, plan.idesc, kb != first || k != 0 ? 1u : 0u);
                mma_commit(smem_addr(&empty[stage]));
                if (++stage == C::kStages) stage = 0, phase ^= 1;
            }
            mma_commit(smem_addr(tfull));
            mbar_wait(tfull, 0, p.status);
        }
    }
    // The join below has one thread per 8 outputs of some tokens: its outputs' vectors, loaded while the products run.
    const int64_t n = n0 + threadIdx.x % (kLanes / 8) * 8;
    float *scales = reinterpret_cast<float *>(smem + C::kScales);
    float4 ws[2] = {}, bias[2] = {};
    if (n < p.out_features) {
        if (E4M3) ws[0] = vector4(p.weight_scale, n, p.out_features, plan.vectors),
                  ws[1] = vector4(p.weight_scale, n + 4, p.out_features, plan.vectors);
        if (p.bias != nullptr) bias[0] = vector4(p.bias, n, p.out_features, plan.vectors),
                               bias[1] = vector4(p.bias, n + 4, p.out_features, plan.vectors);
    }
    if (E4M3 && threadIdx.x < BT && t0 + threadIdx.x < p.num_tokens) scales[threadIdx.x] = p.x_scale[t0 + threadIdx.x];
    __syncwarp();
    // CTA s of the cluster joins tokens [T s / splits, T (s + 1) / splits) of the tile's T.
    const int tokens = static_cast<int>(min(static_cast<int64_t>(BT), p.num_tokens - t0));
    if (SEND) cluster_wait();   // every CTA has started, so its memory may be written
    if (warp < 4) {
        mbar_wait(tfull, 0, p.status, abort_word);
        tc_fence_after();
        const int channel = warp * 32 + lane;
        int owner = 0, first_owned = 0, end_owned = tokens / splits;
#pragma unroll 1
        for (int c = 0; c < tokens; c += 16) {
            uint32_t acc[16];
            tmem_load16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, acc);
            tmem_wait_load();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (SEND) {
                    // Row (token of its owner, split) of the owner's inbox.
                    if (c + j >= tokens) break;
                    while (c + j >= end_owned) first_owned = end_owned, ++owner, end_owned = tokens * (owner + 1) / splits;
                    const int at = (c + j - first_owned) * splits + split;
                    store_peer(peer_addr(base + C::kSums + (at * kLanes + channel) * 4, owner), acc[j]);
                } else {
                    // Every product of this CTA is complete: its stages are free.
                    reinterpret_cast<uint32_t *>(smem + C::kSums)[(c + j) * kLanes + channel] = acc[j];
                }
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    cluster_sync();   // of one CTA too (splits == 1): a block barrier
    if (warp == 5) {
        tc_fence_after();
        tmem_free<1>(tmem, C::kColumns);
    }
    // The sums are joined always in the order of the splits.
    const int from = tokens * split / splits, to = tokens * (split + 1) / splits;
    const uint32_t octet = threadIdx.x % (kLanes / 8) * 32;
    const O *residual = static_cast<const O *>(p.residual);
    O *out = static_cast<O *>(p.out);
    const int count = static_cast<int>(min(static_cast<int64_t>(8), p.out_features - n));
    const bool wide = count == 8 && plan.out_tma && (residual == nullptr || plan.residual_tma);
#pragma unroll 2
    for (int r = from + static_cast<int>(threadIdx.x) / (kLanes / 8); r < to && count > 0; r += C::kThreads / (kLanes / 8)) {
        const int64_t t = t0 + r;
        O *to_row = out + t * p.out_row_stride + n;
        const O *from_row = residual != nullptr ? residual + t * p.residual_row_stride + n : nullptr;
        uint4 res = {};
        if (wide && residual != nullptr) res = *reinterpret_cast<const uint4 *>(from_row);
        float2 y[4] = {};
        for (int s = 0; s < splits; ++s) {
            float4 lo, hi;
            if (SEND) {
                const uint8_t *at = smem + C::kSums + ((r - from) * splits + s) * (kLanes * 4) + octet;
                lo = *reinterpret_cast<const float4 *>(at), hi = *reinterpret_cast<const float4 *>(at + 16);
            } else {
                const uint32_t at = peer_addr(base + C::kSums + r * (kLanes * 4) + octet, s);
                lo = load_peer(at), hi = load_peer(at + 16);
            }
            y[0] = add2(y[0], make_float2(lo.x, lo.y)), y[1] = add2(y[1], make_float2(lo.z, lo.w));
            y[2] = add2(y[2], make_float2(hi.x, hi.y)), y[3] = add2(y[3], make_float2(hi.z, hi.w));
        }
        if (E4M3) {
            const float2 sx = make_float2(scales[r], scales[r]);
            y[0] = mul2(mul2(y[0], make_float2(ws[0].x, ws[0].y)), sx), y[1] = mul2(mul2(y[1], make_float2(ws[0].z, ws[0].w)), sx);
            y[2] = mul2(mul2(y[2], make_float2(ws[1].x, ws[1].y)), sx), y[3] = mul2(mul2(y[3], make_float2(ws[1].z, ws[1].w)), sx);
        }
        y[0] = add2(y[0], make_float2(bias[0].x, bias[0].y)), y[1] = add2(y[1], make_float2(bias[0].z, bias[0].w));
        y[2] = add2(y[2], make_float2(bias[1].x, bias[1].y)), y[3] = add2(y[3], make_float2(bias[1].z, bias[1].w));
        activate_all(p.activation, y);
        if (wide) {
            if (residual != nullptr) {
                y[0] = add2(y[0], unpack2<O>(res.x)), y[1] = add2(y[1], unpack2<O>(res.y));
                y[2] = add2(y[2], unpack2<O>(res.z)), y[3] = add2(y[3], unpack2<O>(res.w));
            }
            *reinterpret_cast<uint4 *>(to_row) = make_uint4(pack2<O>(y[0].x, y[0].y), pack2<O>(y[1].x, y[1].y),
                                                            pack2<O>(y[2].x, y[2].y), pack2<O>(y[3].x, y[3].y));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j >= count) break;
                const float f = (j & 1) != 0 ? y[j / 2].y : y[j / 2].x;
                to_row[j] = from_f32<O>(residual != nullptr ? f + to_f32(from_row[j]) : f);
            }
        }
    }
    if (!SEND) {
        __syncwarp();
        cluster_sync();   // no CTA's sums go away while another reads them
    }
}

// Rows of `columns` elements copied to rows that start on 16 bytes, those of the
// first matrix and then those of the second: a warp per 1024 columns of a row,
// side by side along it, since neither end of a source row is on a boundary.
struct RowCopy {
    const void *src;
    void *dst;
    int64_t src_stride, dst_stride;
    int32_t rows;
};
constexpr int kCopyWarps = 8, kCopyColumns = 1024;

template <typename E>
__global__ void __launch_bounds__(kCopyWarps * 32) realign_kernel(const RowCopy a, const RowCopy b, int32_t columns) {
    let_next_start();
    wait_for_previous();
    int64_t row = static_cast<int64_t>(blockIdx.x) * kCopyWarps + (threadIdx.x >> 5);
    if (row >= static_cast<int64_t>(a.rows) + b.rows) return;
    const bool second = row >= a.rows;
    const RowCopy &c = second ? b : a;
    if (second) row -= a.rows;
    const E *from = static_cast<const E *>(c.src) + row * c.src_stride;
    E *to = static_cast<E *>(c.dst) + row * c.dst_stride;
    const int end = min(columns, (static_cast<int>(blockIdx.y) + 1) * kCopyColumns);
    for (int i = blockIdx.y * kCopyColumns + (threadIdx.x & 31); i < end; i += 8 * 32) {
        E v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * 32 < end) v[j] = from[i + j * 32];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * 32 < end) to[i + j * 32] = v[j];
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int element_bytes(int32_t dtype) { return dtype == KDA_DTYPE_E4M3 ? 1 : 2; }

// Whether TMA can address `rows` rows of `columns` elements at this base and stride.
bool tma_rows(const void *base, int64_t stride, int64_t rows, int64_t columns, int bytes) {
    if ((reinterpret_cast<uintptr_t>(base) & 15u) != 0) return false;
    return rows <= 1 || (stride >= columns && stride * bytes % 16 == 0 && stride < (INT64_C(1) << 39));
}
// A stride for the map of rows that are TMA rows (a single row's stride is never used).
int64_t map_stride(int64_t stride, int64_t rows, int64_t columns, int bytes) {
    return rows > 1 ? stride * bytes : (columns * bytes + 15) / 16 * 16;
}
int64_t padded_columns(const KdaLinearArgs &a) {
    const int64_t per = 16 / element_bytes(a.in_dtype);
    return (a.in_features + per - 1) / per * per;
}
size_t copy_bytes(const KdaLinearArgs &a, int64_t rows) {
    return (static_cast<size_t>(rows) * padded_columns(a) * element_bytes(a.in_dtype) + 255) / 256 * 256;
}
bool copies_x(const KdaLinearArgs &a) {
    return !tma_rows(a.x, a.x_row_stride, a.num_tokens, a.in_features, element_bytes(a.in_dtype));
}
bool copies_weight(const KdaLinearArgs &a) {
    return !tma_rows(a.weight, a.weight_row_stride, a.out_features, a.in_features, element_bytes(a.in_dtype));
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, resolved once through the runtime (the library does not link libcuda).
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return static_cast<EncodeTiled>(nullptr);
        return reinterpret_cast<EncodeTiled>(ptr);
    }();
    return fn;
}

// [rows][columns] with boxes of 128 bytes x box_rows in the 128-byte swizzle; reads past the ends give zeros.
bool encode(CUtensorMap *map, const void *base, int32_t dtype, int64_t rows, int64_t columns, int64_t stride_bytes,
            int box_rows) {
    const EncodeTiled fn = encode_tiled();
    if (fn == nullptr) return false;
    const CUtensorMapDataType type = dtype == KDA_DTYPE_E4M3   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : dtype == KDA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(kRowBytes / element_bytes(dtype)), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t steps[2] = {1, 1};
    return fn(map, type, 2, const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Few tokens: the narrow kernel with the smallest token tile whose tiles fit
// one per SM, then K split until two CTAs per SM are busy (each with 4 blocks
// of K at least). Measured, us (bf16, K = 4096; tile/splits): 64 tokens, N =
// 4096: 16/2 13.0, 64/4 15.0, pair 18.5; 128 tokens: 32/2 14.4, 16/1 18.2, 64/2
// 16.4, pair 18.8; 256 tokens: 64/2 16.5, 32/1 19.9, pair 19.2; N = 12576, 64
// tokens: 64/2 23.6, 32/1 26.5, pair 25.4; 128 tokens: 64/1 29.6, pair 27.8.
// Otherwise the pair kernel, with the width whose waves of tiles take the
// fewest cycles: per tile either its K blocks (measured: 345, 345, 425 and 525
// cycles at widths 64..256) or its epilogue, whichever is longer. What an epilogue
// takes depends on what is in it (measured at K = 64, bf16, widths 64..256: 2,160 to
// 3,070 cycles with none, 3,510 to 5,700 with bias and sigmoid, 4,180 to 10,100 with a
// residual beside); the rule has one figure, between the first two. 256 tokens,
// N = 12576, K = 4096 e4m3: width 192 (66 tiles) 17.7 us, 256 (50) 19.3, 128 (99)
// 23.9; 512 tokens, N = 4096 bf16: 128 (64 tiles) 21.7, 256 (32) 27.0.
KdaLinearForm choose(const KdaLinearArgs &a, int64_t k_blocks, int64_t sms) {
    const int64_t T = a.num_tokens, outputs = (static_cast<int64_t>(a.out_features) + kLanes - 1) / kLanes;
    const int64_t pairs = sms > 1 ? sms / 2 : 1;
    for (int tile = 16; tile <= 64; tile *= 2) {
        const int64_t ctas = outputs * ((T + tile - 1) / tile);
        if (ctas > sms && (T > 64 || tile < T)) continue;
        int64_t splits = 2 * sms / ctas;
        if (splits > k_blocks / 4) splits = k_blocks / 4;
        if (splits > 8) splits = 8;
        return {KDA_LINEAR_NARROW, tile, splits > 1 ? static_cast<int32_t>(splits) : 1};
    }
    static constexpr int kBlockCycles[4] = {345, 345, 425, 525};
    KdaLinearForm best = {KDA_LINEAR_PAIR, 256, 1};
    int64_t least = INT64_MAX;
    for (int i = 3; i >= 0; --i) {
        const int width = 64 * (i + 1);
        const int64_t tiles = (T + Pair::kTileT - 1) / Pair::kTileT * ((a.out_features + width - 1) / width);
        const int64_t products = k_blocks * kBlockCycles[i], epilogue = 2600 + 6 * width;
        const int64_t cycles = (tiles + pairs - 1) / pairs * (products > epilogue ? products : epilogue);
        if (cycles < least) least = cycles, best.tile = width;
    }
    return best;
}

int k_blocks_of(const KdaLinearArgs &a) {
    const int per = kRowBytes / element_bytes(a.in_dtype);
    return (a.in_features + per - 1) / per;
}
// Whether any arguments of `k_blocks` may be launched in this form.
bool form_ok(const KdaLinearArgs &a, int k_blocks, const KdaLinearForm &f) {
    if (f.kernel == KDA_LINEAR_PAIR) return f.splits == 1 && f.tile >= 64 && f.tile <= Pair::kMaxN && f.tile % 64 == 0;
    return f.kernel == KDA_LINEAR_NARROW && (f.tile == 16 || f.tile == 32 || f.tile == 64) && f.splits >= 1 && f.splits <= 8 &&
           f.splits <= k_blocks && (a.num_tokens + f.tile - 1) / f.tile <= 65535;   // the grid's second dimension
}

template <typename O, bool E4M3, bool TMA_ROWS>
cudaError_t launch_pair(const KdaLinearArgs &a, const Plan &plan, const Maps &maps, cudaStream_t st) {
    static OptIn opted;
    if (!opt_in(pair_kernel<O, E4M3, TMA_ROWS>, opted, Pair::kBytes)) return cudaErrorInvalidValue;
    const int64_t tiles = static_cast<int64_t>(plan.tiles_t) * plan.tiles_n;
    const int most = sm_count() > 1 ? sm_count() / 2 : 1, pairs = static_cast<int>(tiles < most ? tiles : most);
    return launch_overlapped(pair_kernel<O, E4M3, TMA_ROWS>, dim3(2 * pairs), Pair::kThreads, Pair::kBytes, 2, st, a, plan, maps);
}

template <typename O, bool E4M3, int BT, bool SEND>
cudaError_t launch_narrow(const KdaLinearArgs &a, const Plan &plan, int splits, const Maps &maps, cudaStream_t st) {
    using C = Narrow<BT, SEND>;
    static OptIn opted;
    if (!opt_in(narrow_kernel<O, E4M3, BT, SEND>, opted, C::kBytes)) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(plan.tiles_n * splits), static_cast<unsigned>(plan.tiles_t));
    return launch_overlapped(narrow_kernel<O, E4M3, BT, SEND>, grid, C::kThreads, C::kBytes, splits, st, a, plan, splits, maps);
}

template <typename O, bool E4M3>
cudaError_t launch_form(const KdaLinearArgs &a, Plan plan, const KdaLinearForm &c, const Maps &maps, cudaStream_t st) {
    const uint32_t format = a.in_dtype == KDA_DTYPE_BF16 ? 1 : 0;
    const bool pair = c.kernel == KDA_LINEAR_PAIR;
    plan.idesc = pair ? instruction_desc(256, c.tile, format) : instruction_desc(kLanes, c.tile, format);
    plan.width = c.tile;
    plan.tail = (a.out_features - (plan.tiles_n - 1) * c.tile + 31) / 32 * 32;
    plan.idesc_tail = instruction_desc(256, plan.tail, format);
    if (pair) {
        const bool tma_rows = plan.out_tma && (a.residual == nullptr || plan.residual_tma);
        return tma_rows ? launch_pair<O, E4M3, true>(a, plan, maps, st) : launch_pair<O, E4M3, false>(a, plan, maps, st);
    }
    if (c.tile == 16)
        return c.splits > 1 ? launch_narrow<O, E4M3, 16, true>(a, plan, c.splits, maps, st)
                            : launch_narrow<O, E4M3, 16, false>(a, plan, c.splits, maps, st);
    if (c.tile == 32) return launch_narrow<O, E4M3, 32, false>(a, plan, c.splits, maps, st);
    return launch_narrow<O, E4M3, 64, false>(a, plan, c.splits, maps, st);
}

int check(const KdaLinearArgs *args) {
    if (args == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    const KdaLinearArgs &a = *args;
    if (a.num_tokens < 0 || a.in_features < 1 || a.out_features < 0) return KDA_ERR_INVALID_ARGUMENT;
    if (a.in_dtype < KDA_DTYPE_BF16 || a.in_dtype > KDA_DTYPE_E4M3) return KDA_ERR_UNSUPPORTED;
    if (a.out_dtype != KDA_DTYPE_BF16 && a.out_dtype != KDA_DTYPE_FP16) return KDA_ERR_UNSUPPORTED;
    if (a.in_dtype != KDA_DTYPE_E4M3 && a.in_dtype != a.out_dtype) return KDA_ERR_UNSUPPORTED;
    if (a.activation < KDA_ACT_NONE || a.activation > KDA_ACT_GELU_TANH) return KDA_ERR_UNSUPPORTED;
    if (a.num_tokens == 0 || a.out_features == 0) return KDA_OK;
    if (a.x == nullptr || a.weight == nullptr || a.out == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    const bool scaled = a.in_dtype == KDA_DTYPE_E4M3;
    if ((a.x_scale != nullptr) != scaled || (a.weight_scale != nullptr) != scaled) return KDA_ERR_INVALID_ARGUMENT;
    if (a.x_row_stride < 0 || a.weight_row_stride < 0 || a.residual_row_stride < 0) return KDA_ERR_INVALID_ARGUMENT;
    if (a.num_tokens > 1 && a.out_row_stride < a.out_features) return KDA_ERR_INVALID_ARGUMENT;
    // Row and column numbers, a tile past the end included, and tile counts stay in int32.
    if (static_cast<int64_t>(a.num_tokens) + a.out_features > INT32_MAX - 512 || a.in_features > 65535 * kCopyColumns)
        return KDA_ERR_TOO_LARGE;
    if ((static_cast<int64_t>(a.num_tokens) / 16 + 1) * (a.out_features / 128 + 1) > INT32_MAX / 16) return KDA_ERR_TOO_LARGE;
    return KDA_OK;
}

size_t workspace_bytes_of(const KdaLinearArgs &a) {
    return (copies_x(a) ? copy_bytes(a, a.num_tokens) : 0) + (copies_weight(a) ? copy_bytes(a, a.out_features) : 0);
}

// In the form given, or the one that choose() takes where it is null.
int launch(const KdaLinearArgs *args, void *workspace, size_t workspace_bytes, const KdaLinearForm *form, cudaStream_t st) {
    const int rc = check(args);
    if (rc != KDA_OK || args->num_tokens == 0 || args->out_features == 0) return rc;
    KdaLinearArgs a = *args;
    const int k_blocks = k_blocks_of(a);
    const KdaLinearForm c = form != nullptr ? *form : choose(a, k_blocks, sm_count());
    if (!form_ok(a, k_blocks, c)) return KDA_ERR_INVALID_ARGUMENT;
    const size_t need = workspace_bytes_of(*args);
    if (need > 0) {
        if (workspace == nullptr || workspace_bytes < need) return KDA_ERR_WORKSPACE;
        if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return KDA_ERR_ALIGNMENT;
        uint8_t *at = static_cast<uint8_t *>(workspace);
        RowCopy copies[2] = {};
        if (copies_x(*args)) {
            copies[0] = {a.x, at, a.x_row_stride, padded_columns(a), a.num_tokens};
            a.x = at;
            a.x_row_stride = padded_columns(a);
            at += copy_bytes(a, a.num_tokens);
        }
        if (copies_weight(*args)) {
            copies[1] = {a.weight, at, a.weight_row_stride, padded_columns(a), a.out_features};
            a.weight = at;
            a.weight_row_stride = padded_columns(a);
        }
        const int64_t rows = static_cast<int64_t>(copies[0].rows) + copies[1].rows;
        const dim3 grid(static_cast<unsigned>((rows + kCopyWarps - 1) / kCopyWarps),
                        static_cast<unsigned>((a.in_features + kCopyColumns - 1) / kCopyColumns));
        const int threads = kCopyWarps * 32;
        const cudaError_t e =
            a.in_dtype == KDA_DTYPE_E4M3
                ? launch_overlapped(realign_kernel<uint8_t>, grid, threads, 0, 1, st, copies[0], copies[1], a.in_features)
                : launch_overlapped(realign_kernel<uint16_t>, grid, threads, 0, 1, st, copies[0], copies[1], a.in_features);
        if (e != cudaSuccess) return KDA_ERR_LAUNCH;
    }
    const int es = element_bytes(a.in_dtype);
    Plan plan = {};
    plan.k_blocks = k_blocks;
    const bool pair = c.kernel == KDA_LINEAR_PAIR;
    const int tile_t = pair ? 256 : c.tile, tile_n = pair ? c.tile : kLanes;
    plan.tiles_t = (a.num_tokens + tile_t - 1) / tile_t;
    plan.tiles_n = (a.out_features + tile_n - 1) / tile_n;
    // A TMA store ends on 16 bytes: past a width that is no multiple of them it would write zeros into what lies
    // beside the row (a store of 3 columns wrote 8). The narrow kernel stores whole vectors inside the row only.
    plan.out_tma = tma_rows(a.out, a.out_row_stride, a.num_tokens, a.out_features, 2) && (!pair || a.out_features % 8 == 0);
    plan.residual_tma =
        a.residual != nullptr && tma_rows(a.residual, a.residual_row_stride, a.num_tokens, a.out_features, 2);
    plan.vectors = ((reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.weight_scale)) & 15u) == 0;
    Maps maps = {};
    bool ok = encode(&maps.x, a.x, a.in_dtype, a.num_tokens, a.in_features,
                     map_stride(a.x_row_stride, a.num_tokens, a.in_features, es), pair ? kLanes : c.tile) &&
              encode(&maps.weight, a.weight, a.in_dtype, a.out_features, a.in_features,
                     map_stride(a.weight_row_stride, a.out_features, a.in_features, es), pair ? c.tile / 2 : kLanes);
    if (pair && plan.out_tma)
        ok = ok && encode(&maps.out, a.out, a.out_dtype, a.num_tokens, a.out_features,
                          map_stride(a.out_row_stride, a.num_tokens, a.out_features, 2), 32);
    if (pair && plan.residual_tma)
        ok = ok && encode(&maps.residual, a.residual, a.out_dtype, a.num_tokens, a.out_features,
                          map_stride(a.residual_row_stride, a.num_tokens, a.out_features, 2), 32);
    if (!ok) return KDA_ERR_LAUNCH;
    cudaError_t e;
    if (a.in_dtype == KDA_DTYPE_BF16)
        e = launch_form<__nv_bfloat16, false>(a, plan, c, maps, st);
    else if (a.in_dtype == KDA_DTYPE_FP16)
        e = launch_form<__half, false>(a, plan, c, maps, st);
    else if (a.out_dtype == KDA_DTYPE_BF16)
        e = launch_form<__nv_bfloat16, true>(a, plan, c, maps, st);
    else
        e = launch_form<__half, true>(a, plan, c, maps, st);
    return e == cudaSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // namespace linear
}  // namespace kda

extern "C" size_t kda_linear_workspace_bytes(const KdaLinearArgs *args) {
    using namespace kda::linear;
    if (check(args) != KDA_OK || args->num_tokens == 0 || args->out_features == 0) return 0;
    return workspace_bytes_of(*args);
}

extern "C" int kda_linear_launch(const KdaLinearArgs *args, void *workspace, size_t workspace_bytes, void *stream) {
    return kda::linear::launch(args, workspace, workspace_bytes, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int kda_linear_form(const KdaLinearArgs *args, int32_t sms, KdaLinearForm *form) {
    using namespace kda::linear;
    const int rc = check(args);
    if (rc != KDA_OK) return rc;
    if (sms < 0 || form == nullptr || args->num_tokens == 0 || args->out_features == 0) return KDA_ERR_INVALID_ARGUMENT;
    *form = choose(*args, k_blocks_of(*args), sms > 0 ? sms : kda::sm_count());
    return KDA_OK;
}

extern "C" int kda_linear_launch_form(const KdaLinearArgs *args, void *workspace, size_t workspace_bytes,
                                      const KdaLinearForm *form, void *stream) {
    if (form == nullptr) return KDA_ERR_INVALID_ARGUMENT;
    return kda::linear::launch(args, workspace, workspace_bytes, form, static_cast<cudaStream_t>(stream));
}
