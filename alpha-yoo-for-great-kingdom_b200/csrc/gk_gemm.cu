// gk_gemm.cu - 16-bit matrix products on tcgen05 with a fused epilogue.
//
// Operands go from global to shared memory by TMA as 128-byte-swizzled panels
// of 64 contiguous elements, whichever of the two dimensions is contiguous:
//   k contiguous:      one panel of (tile rows) x 64 k, 128 bytes a row;
//   m or n contiguous: a panel of 64 k rows for every 64 of m or n.
// The matrix descriptors and the instruction descriptor carry the difference,
// so the forward product (k, k), the input gradient (k, across) and the weight
// gradient (across, across) run in the same kernels. TMA fills what lies
// outside a tensor with zeros, so no size has to be a multiple of anything.
//
// Accumulation is fp32 in TMEM; bias, residual and activation are applied in
// fp32 and each output is rounded once.
#include "gk_gemm.cuh"

#include <cooperative_groups.h>
#include <cuda.h>

#include <cmath>

#include "../../include/gk.h"
#include "gk_act.cuh"
#include "gk_launch.cuh"
#include "gk_tc.cuh"

namespace gk {
namespace {

namespace cg = cooperative_groups;
using namespace tc;

constexpr int kBK = 64;  // k elements of a stage: one 128-byte swizzled row
// An operand's `across` in here: its panels of 64 m or n loaded one by one, or
// all of a stage by one box of a map [panel, k, 64], for sizes that are whole
// panels (dW of 8192 x 4096 -> 8192: 377 -> 357 us).
constexpr int kPanels = 2;

struct Epilogue {
    void* out;
    const void* bias;
    const void* residual;
    void* pre;
    int64_t out_ld, residual_ld, pre_ld;
    int m, n;
    int activation;
    int bf16;
    int out_wide, pre_wide, residual_wide, bias_wide;  // every row (the bias) starts on 16 bytes
};

// Issue is warp-wide: every lane of a converged warp runs the loops, so that
// addresses and descriptors stay on the uniform datapath, and a predicate from
// one elect.sync lets one lane issue. A single thread in a branch of its own
// took about 750 cycles for a stage, half as long again as its MMAs; an
// elect.sync for each instruction about 480.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, e;\n\t}"
        : "=r"(r));
    return r;
}
template <bool PAIR>  // PAIR: the bytes are counted by a barrier of the pair's even CTA
__device__ __forceinline__ void tma_load(uint32_t one, uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint32_t bar) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred e;\n\t"
            "setp.ne.b32 e, %5, 0;\n\t"
            "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
            "[%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar), "r"(one)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred e;\n\t"
            "setp.ne.b32 e, %5, 0;\n\t"
            "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar), "r"(one)
            : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t one, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b64 st;\n\t"
        "setp.ne.b32 e, %2, 0;\n\t"
        "@e mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar),
        "r"(bytes), "r"(one)
        : "memory");
}

// Descriptor of a 128-byte-swizzled operand whose panels start on 1024 bytes.
// k contiguous: rows in groups of 8, 1024 bytes apart. m or n contiguous: k in
// groups of 8 rows, 1024 bytes apart, and panels of 64 m or n, 8192 apart.
// The low word holds the address and the panel step, the high word is the same for all.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, int across) {
    return ((addr & 0x3FFFFu) >> 4) | ((across ? 8192u >> 4 : 1u) << 16);
}
// Address step of 16 k elements, in 16-byte units.
__device__ __forceinline__ uint32_t k_step(int across) { return across ? 16 * 128 / 16 : 32 / 16; }

// The four MMAs of a stage (64 k) and the commit that frees the stage.
template <bool PAIR>
__device__ __forceinline__ void mma_stage(uint32_t one, uint32_t acc, uint32_t a, uint32_t b, uint32_t step_a, uint32_t step_b,
                                          uint32_t idesc, uint32_t accumulate, uint32_t bar) {
#define GK_MMA_STAGE(GROUP, COMMIT)                                                          \
    asm volatile(                                                                            \
        "{\n\t.reg .pred p, e;\n\t.reg .b64 ad, bd;\n\t.reg .b32 al, bl;\n\t"                  \
        "setp.ne.b32 p, %6, 0;\n\t"                                                           \
        "setp.ne.b32 e, %10, 0;\n\t"                                                          \
        "mov.b64 ad, {%1, %8};\n\tmov.b64 bd, {%2, %8};\n\t"                                   \
        "@e tcgen05.mma." GROUP ".kind::f16 [%0], ad, bd, %5, p;\n\t"                          \
        "add.u32 al, %1, %3;\n\tadd.u32 bl, %2, %4;\n\t"                                       \
        "mov.b64 ad, {al, %8};\n\tmov.b64 bd, {bl, %8};\n\t"                                   \
        "@e tcgen05.mma." GROUP ".kind::f16 [%0], ad, bd, %5, 1;\n\t"                          \
        "add.u32 al, al, %3;\n\tadd.u32 bl, bl, %4;\n\t"                                       \
        "mov.b64 ad, {al, %8};\n\tmov.b64 bd, {bl, %8};\n\t"                                   \
        "@e tcgen05.mma." GROUP ".kind::f16 [%0], ad, bd, %5, 1;\n\t"                          \
        "add.u32 al, al, %3;\n\tadd.u32 bl, bl, %4;\n\t"                                       \
        "mov.b64 ad, {al, %8};\n\tmov.b64 bd, {bl, %8};\n\t"                                   \
        "@e tcgen05.mma." GROUP ".kind::f16 [%0], ad, bd, %5, 1;\n\t"                          \
        "@e " COMMIT "\n\t}" ::"r"(acc),                                                       \
        "r"(a), "r"(b), "r"(step_a), "r"(step_b), "r"(idesc), "r"(accumulate), "r"(bar), "r"(kDescHigh), \
        "h"((uint16_t)3), "r"(one)                                                            \
        : "memory")
    if (PAIR)
        GK_MMA_STAGE("cta_group::2",
                     "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%7], %9;");
    else
        GK_MMA_STAGE("cta_group::1", "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];");
#undef GK_MMA_STAGE
}
// Arrives once the MMAs issued so far complete; PAIR: on the barrier at this offset in both CTAs.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred e;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
                bar),
            "h"((uint16_t)3)
            : "memory");
    else
        mma_commit_warp(bar);
}

__host__ __device__ constexpr uint32_t idesc16(int m, int n, int bf16, int a_across, int b_across) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)a_across << 15) |
           ((uint32_t)b_across << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <bool PAIR>  // from (k, panel) of a map of panels
__device__ __forceinline__ void tma_load_panels(uint32_t one, uint32_t dst, const CUtensorMap* map, int k, int panel,
                                                uint32_t bar) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred e;\n\t"
            "setp.ne.b32 e, %6, 0;\n\t"
            "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
            "[%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst),
            "l"(map), "r"(0), "r"(k), "r"(panel), "r"(bar), "r"(one)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred e;\n\t"
            "setp.ne.b32 e, %6, 0;\n\t"
            "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(dst),
            "l"(map), "r"(0), "r"(k), "r"(panel), "r"(bar), "r"(one)
            : "memory");
}
// Load an operand's ROWS x 64 stage: (mn, k) is its first element.
template <int ROWS, bool PAIR>
__device__ __forceinline__ void load_stage(uint32_t one, uint32_t dst, const CUtensorMap* map, int across, int mn, int k,
                                           uint32_t bar) {
    if (across == kPanels) {
        tma_load_panels<PAIR>(one, dst, map, k, mn / 64, bar);
    } else if (across) {
#pragma unroll
        for (int p = 0; p < ROWS / 64; ++p) tma_load<PAIR>(one, dst + p * 8192, map, mn + 64 * p, k, bar);
    } else {
        tma_load<PAIR>(one, dst, map, k, mn, bar);
    }
}
// Whether the phase is over, without waiting (try_wait may sleep for microseconds).
__device__ __forceinline__ bool mbar_look(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// A wait of the whole warp with one verdict. `ready`: an earlier look at the
// barrier (a look takes some 150 cycles, so each is taken a stage ahead, under
// the issue of the stage before).
__device__ __forceinline__ bool warp_wait(bool ready, uint32_t bar, uint32_t parity, uint32_t* status) {
    if (__all_sync(0xffffffffu, ready)) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status));
}

// ------------------------------------------------------------------ split

// Tiles of 128 x 64, one CTA each; with few tiles a cluster of CTAs shares a
// tile along k. Every CTA of the cluster leaves its fp32 part in its shared
// memory, and each then adds up, in rank order, and finishes a share of the
// tile's rows: no workspace, no atomics, one launch.
//
// THIN: a product of at most 128 rows reads B (the weight) once and is bound by
// that. It runs with the operands exchanged, 128 rows of B to a tile and all
// rows of A beside them, so that a stage is mostly weight and the stages hold
// some 100 KB of it in flight; the accumulator is out^T and is turned through
// shared memory. A load of A takes only the rows there are: boxes that lie mostly
// outside the tensor halved the speed (12 x 4096 x 12288: 55 us, 16 rows 27).
//
// Warp 0 loads, warp 1 issues the MMAs, warps 2-9 drain TMEM (two a quadrant of
// its rows, every other 32 columns each), all finish.
constexpr int kSplitThreads = 320;
constexpr int kSplitSmem = 112 * 1024;  // two CTAs an SM
constexpr int kMostStages = 8;
struct SplitShape {
    int bn;  // rows of the second operand in a tile
    __host__ __device__ int stage_bytes() const { return (128 + bn) * kBK * 2; }
    __host__ __device__ int stages() const {
        const int fit = (kSplitSmem - 1024) / stage_bytes();
        return fit < kMostStages ? fit : kMostStages;
    }
    __host__ __device__ int smem() const { return stages() * stage_bytes() + 1024; }
    // fp32 pitch of the part, [128][bn] or THIN [bn][128]: rows 16 bytes apart modulo the banks
    __host__ __device__ static constexpr int pitch(bool thin) { return (thin ? 128 : 64) + 4; }
};
constexpr int kSplitBN = 64;

// Four neighbours of a row, `count` of which there are (fewer at a row's end).
__device__ __forceinline__ void add4(const void* p, int64_t at, int count, bool wide, float (&v)[4], bool bf16) {
    if (wide && count == 4) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at));
        float lo, hi;
        unpack16(x.x, bf16, lo, hi);
        v[0] += lo, v[1] += hi;
        unpack16(x.y, bf16, lo, hi);
        v[2] += lo, v[3] += hi;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) v[j] += load16(p, at + j, bf16);
    }
}
__device__ __forceinline__ void put4(void* p, int64_t at, int count, bool wide, const float (&v)[4], bool bf16) {
    if (wide && count == 4) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + at) =
            make_uint2(pack16(v[0], v[1], bf16), pack16(v[2], v[3], bf16));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) store16(p, at + j, v[j], bf16);
    }
}
// Bias, residual, activation and stores.
__device__ __forceinline__ void finish4(const Epilogue& ep, int64_t m, int n, float (&v)[4], bool bf16) {
    const int count = min(4, ep.n - n);
    if (ep.bias != nullptr) add4(ep.bias, n, count, ep.bias_wide, v, bf16);
    if (ep.residual != nullptr) add4(ep.residual, m * ep.residual_ld + n, count, ep.residual_wide, v, bf16);
    const bool tanh32 = ep.activation == GK_ACT_TANH;  // keeps its fp32 value, not the sum
    if (ep.pre != nullptr && !tanh32) put4(ep.pre, m * ep.pre_ld + n, count, ep.pre_wide, v, bf16);
    if (ep.activation != GK_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = act_value<true>(v[j], ep.activation);
    }
    if (ep.pre != nullptr && tanh32) {
        float* kept = static_cast<float*>(ep.pre) + m * ep.pre_ld + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) kept[j] = v[j];
    }
    put4(ep.out, m * ep.out_ld + n, count, ep.out_wide, v, bf16);
}

template <bool THIN>
__global__ void __launch_bounds__(kSplitThreads, 2) gemm_split_kernel(const __grid_constant__ CUtensorMap ta,
                                                                   const __grid_constant__ CUtensorMap tb,
                                                                   Epilogue ep, int thin_rows, int tiles_n,
                                                                   int k_blocks, int a_across, int b_across,
                                                                   uint32_t* status) {
    constexpr int kA = 128 * kBK * 2, kPitch = SplitShape::pitch(THIN);
    const SplitShape shape{THIN ? thin_rows : kSplitBN};
    const int count = shape.stages(), stage_bytes = shape.stage_bytes();
    extern __shared__ uint8_t raw[];
    __shared__ alignas(8) uint64_t full[kMostStages], empty[kMostStages], done;
    __shared__ uint32_t tmem_slot;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t stages = smem_u32(base);
    const uint32_t tmem_cols = shape.bn <= 32 ? 32 : shape.bn <= 64 ? 64 : 128;
    const int tile_a = blockIdx.x / tiles_n, a_row0 = tile_a * 128, b_row0 = (blockIdx.x - tile_a * tiles_n) * kSplitBN;
    const int kb0 = (int)((int64_t)rank * k_blocks / ranks), kb1 = (int)((int64_t)(rank + 1) * k_blocks / ranks);

    if (threadIdx.x == 0) {
        for (int s = 0; s < count; ++s) mbar_init(smem_u32(&full[s]), 1), mbar_init(smem_u32(&empty[s]), 1);
        mbar_init(smem_u32(&done), 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        bool ok = true, ready = true;  // the first round finds every stage empty
        int s = 0, turn = 0;
        const uint32_t one = elect_one();
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
            ok = warp_wait(ready, smem_u32(&empty[s]), (turn - 1) & 1, status);
            if (!ok) break;
            const int next = s + 1 == count ? 0 : s + 1, next_turn = next == 0 ? turn + 1 : turn;
            ready = next_turn == 0 || mbar_look(smem_u32(&empty[next]), (next_turn - 1) & 1);
            const uint32_t bar = smem_u32(&full[s]), at = stages + s * stage_bytes;
            expect_tx(one, bar, stage_bytes);
            load_stage<128, false>(one, at, &ta, a_across, a_row0, kb * kBK, bar);
            if constexpr (THIN)  // one box of bn rows, k contiguous
                tma_load<false>(one, at + kA, &tb, kb * kBK, 0, bar);
            else
                load_stage<kSplitBN, false>(one, at + kA, &tb, b_across, b_row0, kb * kBK, bar);
            s = next, turn = next_turn;
        }
        // After a wait that gave up: the copies in flight land before the block may end.
        if (!ok)
            for (int i = max(0, turn * count + s - count); i < turn * count + s; ++i)
                mbar_wait(smem_u32(&full[i % count]), (i / count) & 1, status);
    } else if (warp == 1) {
        const uint32_t idesc = idesc16(128, shape.bn, ep.bf16, a_across != 0, b_across != 0);
        const uint32_t step_a = k_step(a_across), step_b = k_step(b_across);
        const uint32_t a0 = desc_low(stages, a_across), b0 = desc_low(stages + kA, b_across);
        int s = 0, parity = 0;
        bool ready = false;
        const uint32_t one = elect_one();
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!warp_wait(ready, smem_u32(&full[s]), parity, status)) break;
            const int next = s + 1 == count ? 0 : s + 1, next_parity = next == 0 ? parity ^ 1 : parity;
            ready = mbar_look(smem_u32(&full[next]), next_parity);
            tc_fence_after();
            mma_stage<false>(one, tmem, a0 + s * (stage_bytes >> 4), b0 + s * (stage_bytes >> 4), step_a, step_b, idesc,
                             kb > kb0 ? 1u : 0u, smem_u32(&empty[s]));
            s = next, parity = next_parity;
        }
        commit<false>(smem_u32(&done));
    }
    __syncwarp();
    // Everyone waits for the accumulator: the parts overwrite the stages. The verdict is the warp's, which the
    // loads from TMEM need whole. Where it did not come, MMAs may still read the stages: they are left as they are.
    const bool complete = __all_sync(0xffffffffu, mbar_wait(smem_u32(&done), 0, status));
    tc_fence_after();
    float* part = reinterpret_cast<float*>(base);
    if (warp >= 2 && complete) {
        const int quadrant = warp & 3, row = quadrant * 32 + lane;
        for (int c = (warp - 2) / 4 * 32; c < shape.bn; c += 64) {
            float v[32];
            tmem_ld32(tmem + ((uint32_t)(quadrant * 32) << 16) + c, v);
            if constexpr (THIN) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c + i < shape.bn) part[(c + i) * kPitch + row] = v[i];
            } else {
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *reinterpret_cast<float4*>(part + row * kPitch + c + i) =
                        make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            }
        }
    }
    tc_fence_before();
    if (ranks > 1)
        cluster.sync();
    else
        __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, tmem_cols);
    }
    // Each rank finishes its share of the tile, four neighbours of an output row
    // at a time: a warp then reads whole lines of a part (with eight, the reads of
    // other CTAs' shared memory in steps of 32 bytes took twice as long).
    constexpr int kQuads = (THIN ? 128 : kSplitBN) / 4;
    const int m0 = THIN ? 0 : a_row0, n0 = THIN ? a_row0 : b_row0;
    const int work = min(THIN ? shape.bn : 128, ep.m - m0) * kQuads;
    const bool bf16 = ep.bf16 != 0;
    if (ranks == 1) {
        for (int i = threadIdx.x; i < work; i += kSplitThreads) {
            const int r = i / kQuads, c = (i % kQuads) * 4;
            if (n0 + c >= ep.n) continue;
            const float4 x = *reinterpret_cast<const float4*>(part + r * kPitch + c);
            float v[4] = {x.x, x.y, x.z, x.w};
            finish4(ep, m0 + r, n0 + c, v, bf16);
        }
        return;
    }
    const int from = (int)((int64_t)work * rank / ranks), to = (int)((int64_t)work * (rank + 1) / ranks);
    for (int i = from + threadIdx.x; i < to; i += kSplitThreads) {
        const int r = i / kQuads, c = (i % kQuads) * 4;
        if (n0 + c >= ep.n) continue;
        float4 x[8];  // the parts of all ranks in flight
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < ranks) x[k] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part, k) + r * kPitch + c);
        float v[4] = {};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < ranks) v[0] += x[k].x, v[1] += x[k].y, v[2] += x[k].z, v[3] += x[k].w;
        finish4(ep, m0 + r, n0 + c, v, bf16);
    }
    cluster.sync();  // no CTA leaves while another reads its part
}

// ------------------------------------------------------------------- pair

// Tiles of 256 x BN on pairs of CTAs (cta_group::2): each CTA holds 128 rows of
// A and half of B's rows, and the tensor cores of both read both halves, so an
// SM stages half of what a tile of its own would need. Persistent: a pair walks
// the tiles, and two accumulators in TMEM let the epilogue of one tile run
// under the products of the next. Bound by the tensor cores: 8192 x 4096 -> 8192
// bf16 with bias, residual, gelu and the kept sum 405 us (1360 TFLOP/s), dx 325
// (1690), dW 357 (1540, both operands across).
// Warp 0 loads, warp 1 of the even CTA issues the MMAs, warp 2 owns TMEM, warps
// 4-11 are the epilogue: two warps a quadrant of 32 rows, each with half the columns.
constexpr int kPairThreads = 384;
template <int BN>
struct Pair {
    static constexpr int kA = 128 * kBK * 2, kB = BN / 2 * kBK * 2, kStage = kA + kB;
    static constexpr int kStages = BN == 256 ? 6 : 8;
    static constexpr int kPatch = 4096;  // an epilogue warp's 32 rows x 64 outputs
    static constexpr int kSmem = kStages * kStage + 8 * kPatch + 1024;
    static constexpr uint32_t kTmem = 2 * BN;
};

__device__ __forceinline__ uint32_t cluster_address(uint32_t local, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
    return a;
}
__device__ __forceinline__ void arrive_at(uint32_t remote) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
__device__ __forceinline__ void mma_commit_drain(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}

// Tile `id` of a walk down groups of eight tile rows, so that the tiles in
// flight at one time share their operands in L2.
__device__ __forceinline__ void tile_at(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
    constexpr int kGroup = 8;
    const int per_group = kGroup * tiles_n, group = id / per_group, first = group * kGroup;
    const int rows = min(kGroup, tiles_m - first), rest = id - group * per_group;
    tm = first + rest % rows;
    tn = rest / rows;
}

template <int ACT>
__device__ __forceinline__ void activate(float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        if constexpr (ACT == GK_ACT_GELU)
            quick_gelus(v[i], v[i + 1]);
        else
            v[i] = act_value<true>(v[i], ACT), v[i + 1] = act_value<true>(v[i + 1], ACT);
    }
}
__device__ __forceinline__ void activate(float (&v)[32], int act) {
    switch (act) {
        case GK_ACT_RELU: activate<GK_ACT_RELU>(v); break;
        case GK_ACT_TANH: activate<GK_ACT_TANH>(v); break;
        case GK_ACT_GELU: activate<GK_ACT_GELU>(v); break;
        case GK_ACT_SILU: activate<GK_ACT_SILU>(v); break;
        default: break;
    }
}

// A patch is 32 rows of 128 bytes whose 16-byte chunks are swizzled by the row,
// as TMA's 128-byte swizzle lays them: no bank conflict by rows or by columns.
__device__ __forceinline__ uint4* patch_chunk(uint8_t* patch, int row, int chunk) {
    return reinterpret_cast<uint4*>(patch + row * 128 + ((chunk ^ (row & 7)) << 4));
}
// This lane's row, columns [32 half, 32 half + 32).
__device__ __forceinline__ void put_row(uint8_t* patch, int lane, int half, const float (&v)[32], bool bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *patch_chunk(patch, lane, half * 4 + i) =
            make_uint4(pack16(v[8 * i], v[8 * i + 1], bf16), pack16(v[8 * i + 2], v[8 * i + 3], bf16),
                       pack16(v[8 * i + 4], v[8 * i + 5], bf16), pack16(v[8 * i + 6], v[8 * i + 7], bf16));
}
__device__ __forceinline__ void add_row(const uint8_t* patch, int lane, int half, float (&v)[32], bool bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint4 x = *patch_chunk(const_cast<uint8_t*>(patch), lane, half * 4 + i);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float lo, hi;
            unpack16(w[j], bf16, lo, hi);
            v[8 * i + 2 * j] += lo, v[8 * i + 2 * j + 1] += hi;
        }
    }
}
__device__ __forceinline__ void add_bias(const Epilogue& ep, int n, float (&v)[32], bool bf16) {
    if (ep.bias_wide && n + 32 <= ep.n) {  // every lane reads the same 64 bytes
        const uint4* b = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(ep.bias) + n);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 x = __ldg(b + i);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                unpack16(w[j], bf16, lo, hi);
                v[8 * i + 2 * j] += lo, v[8 * i + 2 * j + 1] += hi;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (n + i < ep.n) v[i] += load16(ep.bias, n + i, bf16);
    }
}
// The warp's patch to rows [row0, row0 + 32), columns [n, n + 64) of an output; TMA clips what lies outside.
__device__ __forceinline__ void store_patch(const CUtensorMap* map, uint8_t* patch, int n, int row0, int lane) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map),
                     "r"(n), "r"(row0), "r"(smem_u32(patch))
                     : "memory");
        bulk_commit();
    }
}
// The patch may be written again once the last store has read it.
__device__ __forceinline__ void patch_free(int lane) {
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
}

// Rows that do not start on 16 bytes, which TMA cannot write: row by row, a
// lane two columns, as 32-bit words that are shifted by one column where a row
// starts between two words.
__device__ __forceinline__ uint32_t* patch_word(uint8_t* patch, int row, int lane) {
    return reinterpret_cast<uint32_t*>(patch_chunk(patch, row, lane >> 2)) + (lane & 3);
}
__device__ __forceinline__ void write_ragged(void* out, int64_t ld, uint8_t* patch, int n, int row0, int rows,
                                             int cols, int lane) {
    __syncwarp();
    uint16_t* base = static_cast<uint16_t*>(out) + row0 * ld + n;
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
        if (r >= rows) break;
        const uint32_t w = *patch_word(patch, r, lane), next = __shfl_down_sync(0xffffffffu, w, 1);
        uint16_t* to = base + r * ld;
        if ((reinterpret_cast<uintptr_t>(to) & 2) == 0) {
            if (2 * lane + 1 < cols)
                *reinterpret_cast<uint32_t*>(to + 2 * lane) = w;
            else if (2 * lane < cols)
                to[2 * lane] = (uint16_t)w;
        } else {
            if (lane == 0) to[0] = (uint16_t)w;
            if (lane < 31 && 2 * lane + 2 < cols)
                *reinterpret_cast<uint32_t*>(to + 2 * lane + 1) = __funnelshift_r(w, next, 16);
            else if (2 * lane + 1 < cols)
                to[2 * lane + 1] = (uint16_t)(w >> 16);
        }
    }
    __syncwarp();
}
__device__ __forceinline__ void keep_row(float* to, int cols, const float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i < cols) to[i] = v[i];
}
__device__ __forceinline__ void read_ragged(const void* from, int64_t ld, uint8_t* patch, int n, int row0, int rows,
                                            int cols, int lane) {
    const uint16_t* base = static_cast<const uint16_t*>(from) + row0 * ld + n + 2 * lane;
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
        const uint32_t lo = r < rows && 2 * lane < cols ? __ldg(base + r * ld) : 0u;
        const uint32_t hi = r < rows && 2 * lane + 1 < cols ? __ldg(base + r * ld + 1) : 0u;
        *patch_word(patch, r, lane) = lo | hi << 16;
    }
}

template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap t_out, const __grid_constant__ CUtensorMap t_pre, Epilogue ep,
                     int tiles_m, int tiles_n, int k_blocks, int a_across, int b_across, uint32_t* status) {
    using P = Pair<BN>;
    extern __shared__ uint8_t raw[];
    __shared__ alignas(8) uint64_t full[P::kStages], empty[P::kStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_slot;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tiles = tiles_m * tiles_n;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t stages = smem_u32(base);

    if (threadIdx.x == 0) {
        for (int s = 0; s < P::kStages; ++s) mbar_init(smem_u32(&full[s]), 1), mbar_init(smem_u32(&empty[s]), 1);
        for (int a = 0; a < 2; ++a) mbar_init(smem_u32(&acc_full[a]), 1), mbar_init(smem_u32(&acc_empty[a]), 16);
        mbar_init(smem_u32(&drain), 1);
        fence_mbar_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(P::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster.sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        int s = 0, turn = 0;
        bool ok = true, ready = true;  // the first round finds every stage empty
        const uint32_t full0 = cluster_address(smem_u32(full), 0), one = elect_one();
        for (int t = pair; t < tiles && ok; t += pairs) {
            int tm, tn;
            tile_at(t, tiles_m, tiles_n, tm, tn);
            const int m0 = tm * 256 + rank * 128, n0 = tn * BN + rank * (BN / 2);
            for (int kb = 0; kb < k_blocks; ++kb) {
                ok = warp_wait(ready, smem_u32(&empty[s]), (turn - 1) & 1, status);
                if (!ok) break;
                const int next = s + 1 == P::kStages ? 0 : s + 1, next_turn = next == 0 ? turn + 1 : turn;
                ready = next_turn == 0 || mbar_look(smem_u32(&empty[next]), (next_turn - 1) & 1);
                const uint32_t at = stages + s * P::kStage, bar = full0 + s * 8;
                if (rank == 0) expect_tx(one, smem_u32(&full[s]), 2 * P::kStage);
                load_stage<128, true>(one, at, &ta, a_across, m0, kb * kBK, bar);
                load_stage<BN / 2, true>(one, at + P::kA, &tb, b_across, n0, kb * kBK, bar);
                s = next, turn = next_turn;
            }
        }
        // After a wait that gave up: the pair's copies in flight land before the blocks may end.
        if (!ok && rank == 0)
            for (int i = max(0, turn * P::kStages + s - P::kStages); i < turn * P::kStages + s; ++i)
                mbar_wait(smem_u32(&full[i % P::kStages]), (i / P::kStages) & 1, status);
    } else if (warp == 1 && rank == 0) {
        const uint32_t idesc = idesc16(256, BN, ep.bf16, a_across != 0, b_across != 0);
        const uint32_t step_a = k_step(a_across), step_b = k_step(b_across);
        const uint32_t a0 = desc_low(stages, a_across), b0 = desc_low(stages + P::kA, b_across);
        int s = 0, parity = 0, n = 0;
        bool ok = true, ready = false;
        const uint32_t one = elect_one();
        for (int t = pair; t < tiles && ok; t += pairs, ++n) {
            const int a = n & 1, use = n >> 1;
            ok = warp_wait(use == 0, smem_u32(&acc_empty[a]), (use - 1) & 1, status);
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem + a * BN;
            for (int kb = 0; kb < k_blocks; ++kb) {
                ok = warp_wait(ready, smem_u32(&full[s]), parity, status);
                if (!ok) break;
                const int next = s + 1 == P::kStages ? 0 : s + 1, next_parity = next == 0 ? parity ^ 1 : parity;
                ready = mbar_look(smem_u32(&full[next]), next_parity);
                tc_fence_after();
                mma_stage<true>(one, acc, a0 + s * (P::kStage >> 4), b0 + s * (P::kStage >> 4), step_a, step_b, idesc,
                                kb > 0 ? 1u : 0u, smem_u32(&empty[s]));
                s = next, parity = next_parity;
            }
            if (ok) commit<true>(smem_u32(&acc_full[a]));
        }
        if (!ok) {  // the MMAs in flight end before TMEM is freed
            mma_commit_drain(smem_u32(&drain));
            mbar_wait(smem_u32(&drain), 0, status);
        }
    } else if (warp >= 4) {
        const int quadrant = warp & 3, half = (warp - 4) >> 2;
        uint8_t* patch = base + P::kStages * P::kStage + (warp - 4) * P::kPatch;
        const bool bf16 = ep.bf16 != 0, tanh32 = ep.activation == GK_ACT_TANH;  // tanh keeps its fp32 value
        int n = 0;
        for (int t = pair; t < tiles; t += pairs, ++n) {
            const int a = n & 1, use = n >> 1;
            int tm, tn;
            tile_at(t, tiles_m, tiles_n, tm, tn);
            const int row0 = tm * 256 + rank * 128 + quadrant * 32, n0 = tn * BN + half * (BN / 2);
            // Every lane waits: the verdict is the warp's.
            if (__any_sync(0xffffffffu, !mbar_wait(smem_u32(&acc_full[a]), use & 1, status))) break;
            tc_fence_after();
            const uint32_t from = tmem + ((uint32_t)(quadrant * 32) << 16) + a * BN + half * (BN / 2);
#pragma unroll 1
            for (int c = 0; c < BN / 2; c += 64) {
                const bool in = row0 < ep.m && n0 + c < ep.n;
                uint4 held[8];
                const bool wide = in && ep.residual != nullptr && ep.residual_wide;
                if (wide) {  // eight lanes a row of 128 bytes, in flight while TMEM is read
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = row0 + i * 4 + (lane >> 3), col = n0 + c + (lane & 7) * 8;
                        held[i] = row < ep.m && col < ep.n
                                      ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(ep.residual) +
                                                                            row * ep.residual_ld + col))
                                      : make_uint4(0, 0, 0, 0);
                    }
                }
                float v0[32], v1[32];
                tmem_ld32x2(from + c, from + c + 32, v0, v1);
                if (c + 64 == BN / 2) {  // the last columns are in registers: the accumulator is free
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_at(cluster_address(smem_u32(&acc_empty[a]), 0));
                }
                if (!in) continue;
                const int rows = min(32, ep.m - row0), cols = min(64, ep.n - n0 - c);
                if (ep.bias != nullptr) {
                    add_bias(ep, n0 + c, v0, bf16);
                    add_bias(ep, n0 + c + 32, v1, bf16);
                }
                patch_free(lane);
                if (ep.residual != nullptr) {
                    if (wide) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) *patch_chunk(patch, i * 4 + (lane >> 3), lane & 7) = held[i];
                    } else {
                        read_ragged(ep.residual, ep.residual_ld, patch, n0 + c, row0, rows, cols, lane);
                    }
                    __syncwarp();
                    add_row(patch, lane, 0, v0, bf16);
                    add_row(patch, lane, 1, v1, bf16);
                }
                if (ep.pre != nullptr && !tanh32) {  // each lane has read its row of the residual and writes the same row
                    put_row(patch, lane, 0, v0, bf16);
                    put_row(patch, lane, 1, v1, bf16);
                    if (ep.pre_wide)
                        store_patch(&t_pre, patch, n0 + c, row0, lane);
                    else
                        write_ragged(ep.pre, ep.pre_ld, patch, n0 + c, row0, rows, cols, lane);
                }
                activate(v0, ep.activation);
                activate(v1, ep.activation);
                if (ep.pre != nullptr && tanh32 && lane < rows) {
                    float* kept = static_cast<float*>(ep.pre) + (row0 + lane) * ep.pre_ld + n0 + c;
                    keep_row(kept, cols, v0);
                    keep_row(kept + 32, cols - 32, v1);
                }
                patch_free(lane);
                put_row(patch, lane, 0, v0, bf16);
                put_row(patch, lane, 1, v1, bf16);
                if (ep.out_wide)
                    store_patch(&t_out, patch, n0 + c, row0, lane);
                else
                    write_ragged(ep.out, ep.out_ld, patch, n0 + c, row0, rows, cols, lane);
            }
        }
        if (lane == 0) bulk_wait<0>();  // the stores are done before the block ends
    }
    __syncwarp();
    tc_fence_before();
    cluster.sync();  // both CTAs are done with the other's barriers, shared memory and TMEM
    tc_fence_after();
    if (warp == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::kTmem) : "memory");
}

// ------------------------------------------------------------------ host

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Map of an operand of `mn` rows (or columns, if across) by k; a box is 64
// contiguous elements by `rows` (k contiguous) or by 64 k (across).
bool encode(CUtensorMap* map, const void* p, int64_t ld, int across, int64_t mn, int64_t k, int rows, int dtype) {
    EncodeFn fn = encoder();
    if (fn == nullptr) return false;
    if (across == kPanels) {
        const cuuint64_t dims[3] = {kBK, (cuuint64_t)k, (cuuint64_t)mn / 64};
        const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, 128};
        const cuuint32_t box[3] = {kBK, kBK, (cuuint32_t)rows / 64};
        const cuuint32_t steps[3] = {1, 1, 1};
        return fn(map, dtype == GK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)(across ? mn : k), (cuuint64_t)(across ? k : mn)};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {kBK, (cuuint32_t)(across ? kBK : rows)};
    const cuuint32_t steps[2] = {1, 1};
    return fn(map, dtype == GK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
              const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

Epilogue epilogue_of(const GemmArgs& g) {
    Epilogue e{g.out, g.bias, g.residual, g.pre, g.out_ld, g.residual_ld, g.pre_ld, (int)g.m, (int)g.n,
               g.activation, g.dtype == GK_BF16, 0, 0, 0, 0};
    e.out_wide = aligned16(g.out) && g.out_ld % 8 == 0;
    e.pre_wide = aligned16(g.pre) && g.pre_ld % 8 == 0;
    // Read in whole 16 bytes, which must not reach past a row: it may be the last of its storage (an expanded one is).
    e.residual_wide = aligned16(g.residual) && g.residual_ld % 8 == 0 && g.n % 8 == 0;
    e.bias_wide = aligned16(g.bias);
    return e;
}

// CTAs that share a tile along k: until they fill two to an SM, in parts of four stages or more.
int split_ranks(int64_t tiles, int64_t stages) {
    int ranks = 1;
    while (ranks < 8 && tiles * ranks * 2 <= 2 * kSmCount && stages >= ranks * 2 * 4) ranks *= 2;
    return ranks;
}

// The same for thin products, of any size up to eight and short of two to an
// SM: clusters of some sizes do not pack the last slots.
int thin_ranks(int64_t tiles, int64_t stages) {
    int64_t ranks = 256 / tiles;
    if (ranks > 8) ranks = 8;
    if (ranks > stages / 4) ranks = stages / 4;
    return ranks < 1 ? 1 : (int)ranks;
}

template <bool THIN>
int launch_split(const GemmArgs& g, uint32_t* status, cudaStream_t stream) {
    auto* kernel = gemm_split_kernel<THIN>;
    static bool ready[64] = {};
    if (!once_per_device(ready, [&] {
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmem) == cudaSuccess;
        }))
        return setup_failed();
    // THIN: the weight is the first operand, and the tile holds all rows of the other.
    const SplitShape shape{THIN ? (int)((g.m + 15) / 16 * 16) : kSplitBN};
    CUtensorMap ta, tb;
    if (THIN ? !encode(&ta, g.b, g.b_ld, g.b_across, g.n, g.k, 128, g.dtype) ||
                   !encode(&tb, g.a, g.a_ld, 0, g.m, g.k, shape.bn, g.dtype)
             : !encode(&ta, g.a, g.a_ld, g.a_across, g.m, g.k, 128, g.dtype) ||
                   !encode(&tb, g.b, g.b_ld, g.b_across, g.n, g.k, shape.bn, g.dtype))
        return GK_EINVAL;
    const int64_t tiles_a = ((THIN ? g.n : g.m) + 127) / 128, tiles_b = THIN ? 1 : (g.n + kSplitBN - 1) / kSplitBN;
    const int64_t blocks = (g.k + kBK - 1) / kBK;
    const int ranks = THIN ? thin_ranks(tiles_a, blocks) : split_ranks(tiles_a * tiles_b, blocks);
    cudaLaunchConfig_t cfg = {};
    if (tiles_a * tiles_b >= (1ll << 31)) return GK_EINVAL;
    cfg.gridDim = dim3((unsigned)(tiles_a * tiles_b), 1, (unsigned)ranks);
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = shape.smem();
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = ranks;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, ta, tb, epilogue_of(g), shape.bn, (int)tiles_b, (int)blocks,
                                   THIN ? g.b_across : g.a_across, THIN ? 0 : g.b_across, status);
}

template <int BN>
int launch_pair(const GemmArgs& g, uint32_t* status, cudaStream_t stream) {
    using P = Pair<BN>;
    auto* kernel = gemm_pair_kernel<BN>;
    static bool ready[64] = {};
    if (!once_per_device(ready, [&] {
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kSmem) == cudaSuccess;
        }))
        return setup_failed();
    const Epilogue ep = epilogue_of(g);
    CUtensorMap ta, tb, t_out = {}, t_pre = {};
    if (!encode(&ta, g.a, g.a_ld, g.a_across, g.m, g.k, 128, g.dtype) ||
        !encode(&tb, g.b, g.b_ld, g.b_across, g.n, g.k, BN / 2, g.dtype))
        return GK_EINVAL;
    // The outputs as [m, n] with n contiguous, in boxes of 64 columns by 32 rows.
    if ((ep.out_wide && !encode(&t_out, g.out, g.out_ld, 0, g.m, g.n, 32, g.dtype)) ||
        (g.pre != nullptr && ep.pre_wide && g.activation != GK_ACT_TANH && !encode(&t_pre, g.pre, g.pre_ld, 0, g.m, g.n, 32, g.dtype)))
        return GK_EINVAL;
    const int64_t tiles_m = (g.m + 255) / 256, tiles_n = (g.n + BN - 1) / BN;
    if (tiles_m * tiles_n >= (1ll << 31) - kSmCount) return GK_EINVAL;
    const int64_t pairs = tiles_m * tiles_n < kSmCount / 2 ? tiles_m * tiles_n : kSmCount / 2;
    kernel<<<(unsigned)(2 * pairs), kPairThreads, P::kSmem, stream>>>(
        ta, tb, t_out, t_pre, ep, (int)tiles_m, (int)tiles_n, (int)((g.k + kBK - 1) / kBK), g.a_across, g.b_across,
        status);
    return launch_status();
}

}  // namespace

int gemm16(const GemmArgs& given, uint32_t* status, cudaStream_t stream) {
    GemmArgs g = given;
    if (g.a_across && g.m % 64 == 0) g.a_across = kPanels;
    if (g.b_across && g.n % 64 == 0) g.b_across = kPanels;
    if (g.m < 1 || g.n < 1 || g.k < 1 || g.m >= (1ll << 31) || g.n >= (1ll << 31) || g.k >= (1ll << 31))
        return GK_EINVAL;
    if (!aligned16(g.a) || !aligned16(g.b) || g.a_ld % 8 != 0 || g.b_ld % 8 != 0) return GK_EINVAL;
    // The form is taken by an estimate of its time in microseconds: a start, and
    // for every round of the tiles that run at once the stages of k that one CTA
    // (or pair) walks, or the epilogue where k is short. Measured
    // (split 128 x 64 | pairs 256 x 128 | pairs 256 x 256; m x k x n):
    // 16 x 4096 x 4096 10.8 | 20.5 | 23.9, 256 x 256 x 256 6.9 | 6.4 | 8.0,
    // 256 x 4096 x 4096 17.0 | 21.5 | 25.3, 1024 x 256 x 4096 14.3 | 8.9 | 8.6,
    // 1024 x 1024 x 1024 10.5 | 9.7 | 11.7, 2048^3 29.5 | 22.7 | 17.8,
    // 4096^3 161 | 123 | 95, 16384 x 1024 x 256 21.2 | 14.8 | 12.5.
    // Up to 64 rows fill half of a split tile, and the estimate takes 1.3 us off it. Where that decides between the
    // forms (split | the pairs that would run instead): 64 x 512 x 128 4.3 | 5.1, 64 x 1024 x 256 4.8 | 5.6,
    // 64 x 4096 x 512 6.3 | 6.7, 49 x 64 x 512 5.5 | 5.9, 49 x 4096 x 512 7.1 | 7.1.
    const double stages = (double)((g.k + kBK - 1) / kBK);
    auto rounds = [](int64_t work, int64_t at_once) { return (double)((work + at_once - 1) / at_once); };
    const int64_t tiles_m = (g.m + 255) / 256, split_tiles = ((g.m + 127) / 128) * ((g.n + 63) / 64);
    const int ranks = split_ranks(split_tiles, (g.k + kBK - 1) / kBK);
    const double split = rounds(split_tiles * ranks, 2 * kSmCount) * (6.3 + stages / ranks * 0.28) -
                         (g.m <= 64 ? 1.3 : 0.0);
    const double narrow = 5.3 + rounds(tiles_m * ((g.n + 127) / 128), kSmCount / 2) * fmax(stages * 0.233, 1.3);
    const double wide = 5.6 + rounds(tiles_m * ((g.n + 255) / 256), kSmCount / 2) * fmax(stages * 0.28, 2.0);
    // The thin form, where the weight's bytes bound the product (thin | best of the
    // others, us; m x k x n): 12 x 4096 x 12288 20.5 | 54, 37 x 8192 x 4096 17.7 | 18.3,
    // 37 x 4096 x 32000 45.5 | 53.5, 64 x 4096 x 4096 13.6 | 12.9, 128 x 4096 x 12288
    // 27.6 | 29.3, 128 x 512 x 16384 13.7 | 11.4, 128 x 4096 x 4096 17.2 | 14.1 (its
    // outputs go through other CTAs' shared memory as often as ranks share a tile).
    if (g.a_across == 0 && (g.m <= 48 || (g.m <= 128 && g.n >= 64 * 128 && g.k >= 1024)))
        return launch_split<true>(g, status, stream);
    if (split <= narrow && split <= wide) return launch_split<false>(g, status, stream);
    return narrow <= wide ? launch_pair<128>(g, status, stream) : launch_pair<256>(g, status, stream);
}

}  // namespace gk
