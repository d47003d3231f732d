// ark_wgrad.cu -- the weight gradient of a projection from its input's 8-bit
// checkpoint:  dW[i, o] (+)= sum over tokens t of X[t, i] * dY[t, o].
//
// Both operands have the summed dimension (tokens) as their slow one, so both
// go to the tensor cores MN-major: a stage holds 64 tokens as rows of 128
// bytes (64 columns), 8 rows to a 1024-byte swizzle atom; accumulators are FP32
// in TMEM.  A byte of X, at most 8 significant bits times a power of two, becomes a
// BF16 operand exactly, and an FP16 one if X was FP16 (operand16).  FP16 dY with a
// checkpoint of a wider type is brought to BF16 operands, whose range holds X: dY as
// the sum of two of them, which holds its 11 bits, and so in two products (wide).
//
// Many tiles (pair_kernel): X is unpacked once into a 16-bit workspace, then
// both operands come by TMA to pairs of CTAs with 256 x 256 tiles.  The grid is
// persistent and two accumulators alternate, so that the epilogue of a tile
// runs under the products of the next one.  Turning the bytes into operands
// inside this kernel was built and measured first: every tile of dY's columns
// turns the same bytes again, and at the power limit each instruction beside
// the products costs clock: 8192 tokens, 4096 x 11008: 640 us against 488 us
// for the products alone.
//
// Few tiles (few_kernel): latency counts, so one launch does it all.  One CTA
// per 128 x 128 tile; 8 of its 14 warps read bytes, turn them in registers and
// store them to the swizzled shape, dY comes by TMA.  The tokens are split over
// a cluster of up to 8 CTAs whose FP32 partial tiles are added over distributed
// shared memory in rank order: no workspace, the same bits every time.
//
// Every wait is bounded.  One that runs out makes its CTA leave NaN in its tiles
// from there on, which the step's finite check turns into a skipped step.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "ark_act8.cuh"
#include "ark_ring.h"

namespace ark {
namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 4, kTeam = 4, kTeams = 2, kCvtWarps = kTeam * kTeams;
constexpr int kThreads = (kEpiWarps + kCvtWarps + 2) * 32;
constexpr int kTmaWarp = kEpiWarps + kCvtWarps, kMmaWarp = kTmaWarp + 1;
constexpr int kPairEpiWarps = 16, kPairThreads = (kPairEpiWarps + 2) * 32;
constexpr int kAtom = kBK * 128;              // 64 tokens x 64 columns of 16 bits
constexpr int kABytes = kBM / 64 * kAtom;
constexpr int kAhead = 2;                     // steps of a team in flight
// The tensor cores add 16 tokens at a time to a sum that is cut off to FP32, not
// rounded: each addition may lose a unit of the last place, 2^-23 of the sum, and
// always towards zero.  So one accumulator takes a bounded run of 64-token steps, and
// runs are added by FP32 additions that round.  FP32 gradients of the pairs: 16 steps,
// 64 additions (4001 tokens of both signs, 2048 x 5504: off by 2.0e-7 in 77.0 us; 32
// steps 4.4e-7 in 76.4, 8 steps 1.1e-7 in 81.5).  16-bit ones: as many as lose an
// eighth of the type's half step, 2^-14 for FP16 (512 additions) and 2^-11 for BF16
// (4096).  Few tiles: up to 32 steps in each of four accumulators.
constexpr uint32_t kRun32 = 16, kRunF16 = 128, kRunBF16 = 1024;
constexpr uint32_t kFewRuns = 4, kFewRun = 32;
constexpr uint32_t kSleepNs = 1000000;
constexpr long long kWaitClocks = 4000000000ll;   // 2 s

struct Few {      // a CTA alone: 128 x 128
    static constexpr int kBN = 128, kBBytes = kBN / 64 * kAtom, kStage = kABytes + kBBytes;
    static constexpr int kStages = 6, kSmem = kStages * kStage + 1024;   // slack to align to 1024
    static constexpr int kRow = kBN + 4;                                 // FP32 row of a partial tile
    static_assert(kBM * kRow * 4 <= kStages * kStage, "partial tile fits the stages");
};
struct Pair {     // two CTAs: 256 x 256, of which each brings 128 columns of dY
    static constexpr int kBN = 256, kBBytes = kBN / 2 / 64 * kAtom, kStage = kABytes + kBBytes;
    static constexpr int kStages = 6, kStaged = 16 * 32 * 16 * 4;   // epilogue: 2 KB per warp
    static constexpr int kSmem = kStages * kStage + kStaged + 1024;
};

struct Out {
    void* p;
    uint64_t ld;
    int f32, bf16, vec;   // vec: rows of whole 16-byte vectors
};

struct Args {
    const uint8_t* x;
    const uint8_t* scale;
    uint64_t pitch, spitch;   // bytes
    uint32_t tokens, m, n;
    uint32_t iters;           // 64-token steps in all
    uint32_t tiles_m, tiles_n, tiles;
    uint32_t chunks;          // runs of steps whose sums are added by the epilogue
    uint32_t splits;          // pair_kernel: runs of tokens that are tiles of their own,
    float* partial;           // and where their FP32 sums go, [splits][m][n_pad], or null
    uint32_t n_pad;
    Out out;
    int accumulate;
};

// ------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The instructions below that one lane issues take their operands from uniform
// registers.  All lanes of the warp run through them and `me` predicates the
// instruction itself: inside a branch on the lane, each operand would be moved to
// a uniform register first, and the issuing lane became the bottleneck (640
// clocks a step, of which the products take 512).
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes, uint32_t me) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
        " @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(bar),
        "r"(bytes), "r"(me)
        : "memory");
}
// one lane of a converged warp
__device__ __forceinline__ uint32_t elect() {
    uint32_t me;
    asm volatile(
        "{\n .reg .pred q;\n elect.sync _|q, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(me));
    return me;
}
// an mbarrier's address in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t bar_of(uint32_t bar, uint32_t rank) {
    uint32_t p;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(bar), "r"(rank));
    return p;
}
// Arrives at a barrier of either CTA of a pair.  What the arrival stands for is
// an SM's own shared memory or TMEM, read by that SM's tensor cores: the writer's
// proxy fence (or tcgen05 fence) before it orders that, and a release at cluster
// scope, which measured 1400 clocks, is not needed for it.
__device__ __forceinline__ void bar_arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// a poll that may sleep for kSleepNs
__device__ __forceinline__ bool bar_sleep(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSleepNs)
        : "memory");
    return ok != 0;
}
// False once the wait has run out, or another warp's has.
enum How { kPoll, kSleep };   // kSleep: for a whole tile
template <How HOW = kPoll>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    long long t0 = 0;   // the clock is not read by a wait that ends soon
    for (uint32_t i = 1;; ++i) {
        if (HOW == kSleep ? bar_sleep(bar, parity) : bar_test(bar, parity)) return true;
        if (HOW == kSleep || (i & 63u) == 0) {
            if (*gave_up) return false;
            const long long now = clock64();
            if (!t0) t0 = now;
            if (now - t0 > kWaitClocks) {
                *gave_up = 1;
                return false;
            }
        }
    }
}
// the same, for what has to be over before a CTA leaves
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!bar_test(bar, parity))
        if (clock64() - t0 > kWaitClocks) break;
}
// the first, for all lanes of a warp
template <How HOW = kPoll>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    return __all_sync(0xFFFFFFFFu, bar_wait<HOW>(bar, parity, gave_up));
}
// PAIR: the barrier may be the other CTA's
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint32_t bar, uint32_t me) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
            " @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3}], [%4];\n}\n" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar), "r"(me)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
            " @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3}], [%4];\n}\n" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar), "r"(me)
            : "memory");
}
// Shared-memory operand, MN-major, 128-byte swizzle: 64-column atoms kAtom
// bytes apart, groups of 8 tokens 1024 bytes apart.  The address field counts 16
// bytes, so operand(at) + bytes / 16 is the operand `bytes` further on.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(kAtom >> 4) << 16 |
           (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// PAIR: a pair of CTAs, M = 256, each CTA holds its 128 rows of A and half of B
template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t add, uint32_t me) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(me)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(me)
            : "memory");
}
// PAIR: arrives at the same barrier of both CTAs
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t me) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
            " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
            "[%0], %1;\n}\n" ::"r"(bar),
            "h"((uint16_t)3), "r"(me)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
                bar),
            "r"(me)
            : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// everything before this grid in the stream is done and visible
__device__ __forceinline__ void wait_before() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ int peer_flag(uint32_t addr, uint32_t rank) {
    uint32_t p;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_ld(uint32_t addr, uint32_t rank) {
    uint32_t p;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(p)
                 : "memory");
    return v;
}

// ------------------------------------------------------------ output
__device__ __forceinline__ float out_get(const Out& o, uint64_t i) {
    if (o.f32) return static_cast<const float*>(o.p)[i];
    if (o.bf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(o.p)[i]);
    return __half2float(static_cast<const __half*>(o.p)[i]);
}
__device__ __forceinline__ void out_put(const Out& o, uint64_t i, float v) {
    if (o.f32)
        static_cast<float*>(o.p)[i] = v;
    else if (o.bf16)
        static_cast<__nv_bfloat16*>(o.p)[i] = __float2bfloat16_rn(v);
    else
        static_cast<__half*>(o.p)[i] = __float2half_rn(v);
}
// four elements of a row of whole vectors
__device__ __forceinline__ void out_old4(const Out& o, uint64_t i, float* v) {
    if (o.f32)
        load_vec<4>(static_cast<const float*>(o.p) + i, v);
    else if (o.bf16)
        load_vec<4>(static_cast<const __nv_bfloat16*>(o.p) + i, v);
    else
        load_vec<4>(static_cast<const __half*>(o.p) + i, v);
}
__device__ __forceinline__ void out_put4(const Out& o, uint64_t i, const float* v) {
    if (o.f32)
        store_vec<4>(static_cast<float*>(o.p) + i, v);
    else if (o.bf16)
        store_vec<4>(static_cast<__nv_bfloat16*>(o.p) + i, v);
    else
        store_vec<4>(static_cast<__half*>(o.p) + i, v);
}
// four sums of one row of an m x n output, rounded once to its type
__device__ __forceinline__ void out_row4(const Out& o, uint32_t m, uint32_t n, uint32_t row,
                                         uint32_t col, float* v, bool accumulate) {
    if (row >= m || col >= n) return;
    const uint64_t i = (uint64_t)row * o.ld + col;
    if (o.vec && col + 4 <= n) {
        float old[4];
        if (accumulate) {
            out_old4(o, i, old);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __fadd_rn(v[j], old[j]);
        }
        out_put4(o, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < n) out_put(o, i + j, accumulate ? __fadd_rn(v[j], out_get(o, i + j)) : v[j]);
    }
}

// A warp's 32 x 16 block of sums, staged in shared memory, to rows row0 on and
// columns col0 on of an m x n output.  Through the staging four lanes come to
// share a row, so that a store fills whole sectors of 8 rows; element by element
// (rows on any boundary) 16 lanes share one.  What is added to is read before any of
// it is written: 2 of a lane's 4 rows at a time, since 4 took registers that the sums
// need (57 tokens, 1117 x 3744 BF16: 10.6 us with 2, 12.4 with 4), and kept as it lies
// there, since widening one waits for it (3741 columns, added: 27 us against 39).
template <class O>
__device__ __forceinline__ void out_block(O* p, const Out& o, uint32_t m, uint32_t n, uint32_t row0,
                                          uint32_t col0, const float4* staged, uint32_t lane,
                                          bool accumulate) {
    using Raw4 = typename std::conditional<sizeof(O) == 4, uint4, uint2>::type;   // four elements
    constexpr int kRows = 2;
    if (o.vec && col0 + 16 <= n) {
        const uint32_t r0 = lane / 4;
        p += (uint64_t)(row0 + r0) * o.ld + col0 + (lane & 3) * 4;
#pragma unroll 1
        for (int h = 0; h < 4; h += kRows) {
            Raw4 old[kRows];
            if (accumulate) {
#pragma unroll
                for (int i = 0; i < kRows; ++i)
                    if (row0 + r0 + (h + i) * 8 < m)
                        old[i] = *reinterpret_cast<const Raw4*>(p + (uint64_t)(i * 8) * o.ld);
            }
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const uint32_t r = r0 + (h + i) * 8;
                const float4 f = staged[r * 4 + ((lane & 3) ^ (r >> 1 & 3))];
                float v[4] = {f.x, f.y, f.z, f.w};
                if (accumulate) {
                    float w[4];
                    load_vec<4>(reinterpret_cast<const O*>(&old[i]), w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = __fadd_rn(v[j], w[j]);
                }
                if (row0 + r < m) store_vec<4>(p + (uint64_t)(i * 8) * o.ld, v);
            }
            p += (uint64_t)(kRows * 8) * o.ld;
        }
        return;
    }
    const uint32_t e = lane & 15, r0 = lane / 16;
    const float* one = reinterpret_cast<const float*>(staged);
    if (col0 + e >= n) return;
    p += (uint64_t)(row0 + r0) * o.ld + col0 + e;
#pragma unroll 1
    for (uint32_t h = 0; h < 32; h += 8, p += 8 * o.ld) {
        O old[4];
        if (accumulate) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row0 + r0 + h + 2 * i < m) old[i] = p[(uint64_t)(2 * i) * o.ld];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = r0 + h + 2 * i;
            float v = one[(r * 4 + (e / 4 ^ (r >> 1 & 3))) * 4 + e % 4];
            if (accumulate) v = __fadd_rn(v, Elem<O>::to_f(old[i]));
            if (row0 + r < m) p[(uint64_t)(2 * i) * o.ld] = Elem<O>::from_f(v);
        }
    }
}

// ------------------------------------------------------------ bytes to a stage
// where part p of n equal ones begins
__device__ __forceinline__ uint32_t part_of(uint32_t total, uint32_t p, uint32_t n) {
    return (uint32_t)((uint64_t)total * p / n);
}

// Teams of 4 warps take steps in turn, so that one's waits, fences and
// instruction latency run under the other's conversions.  A thread turns 16
// bytes (half a scale block) of each of four token rows.
//   col: first column of x of this CTA's tile
template <class T, int KIND, int STAGE, int STAGES>
__device__ __forceinline__ void fill_stages(const Args& a, uint32_t it0, uint32_t it1, uint32_t col,
                                            uint32_t stages, const uint64_t* empty,
                                            const uint64_t* full, volatile int* gave_up) {
    static_assert(STAGES >= kTeams, "a team has a stage of its own");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = (threadIdx.x - kEpiWarps * 32) & (kTeam * 32 - 1);
    const uint32_t team = (warp - kEpiWarps) / kTeam;
    const uint32_t row = t >> 3, unit = t & 7;
    const uint32_t atom = unit >> 2, chunk = (unit & 3) * 2;
    uint4 q[kAhead][4];
    uint32_t sc[kAhead][4];
    // this thread's first row of the step that is loaded next, and where the
    // part's rows end
    uint32_t tok = (it0 + team) * kBK + row;
    const uint32_t end = min(a.tokens, it1 * kBK);
    const uint8_t* xp = a.x + tok * a.pitch + col + unit * 16;
    const uint8_t* sp = a.scale + tok * a.spitch + (col >> 5) + (unit >> 1);
    const uint64_t next_x = kTeams * kBK * a.pitch, next_s = kTeams * kBK * a.spitch;
    auto load = [&](int p) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            q[p][h] = make_uint4(0u, 0u, 0u, 0u);
            sc[p][h] = 127;
            if (tok + 16 * h < end) {
                q[p][h] = __ldg(reinterpret_cast<const uint4*>(xp + h * 16 * a.pitch));
                sc[p][h] = __ldg(sp + h * 16 * a.spitch);
            }
        }
        tok += kTeams * kBK;
        xp += next_x;
        sp += next_s;
    };
#pragma unroll
    for (int p = 0; p < kAhead; ++p) load(p);
    uint32_t todo = (it1 - it0 + kTeams - 1 - team) / kTeams;
    uint32_t s = team, phase = 0;
    bool ok = true;
    while (ok && todo) {
#pragma unroll
        for (int p = 0; p < kAhead; ++p) {
            if (!ok || !todo) break;
            // converted in registers before the stage is free: a stage is held
            // only while it is written
            uint4 lo[4], hi[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) operand16<T, KIND, true>(q[p][h], sc[p][h], lo[h], hi[h]);
            load(p);
            if (!(ok = warp_wait(smem_u32(empty + s), phase ^ 1u, gave_up))) break;
            const uint32_t at = stages + s * STAGE + atom * kAtom;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint32_t r = row + 16 * h;
                // the two atoms' threads store their halves in opposite order: 8
                // neighbouring lanes then cover all 32 banks
                const uint4 one = atom ? hi[h] : lo[h], two = atom ? lo[h] : hi[h];
                const uint32_t base = at + r * 128;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                 base + (((chunk + atom) ^ (r & 7u)) << 4)),
                             "r"(one.x), "r"(one.y), "r"(one.z), "r"(one.w)
                             : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                 base + (((chunk + 1 - atom) ^ (r & 7u)) << 4)),
                             "r"(two.x), "r"(two.y), "r"(two.z), "r"(two.w)
                             : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(full + s));
            s += kTeams;
            if (s >= STAGES) s -= STAGES, phase ^= 1u;
            --todo;
        }
    }
}

// ------------------------------------------------------------ the kernels
// FP32 accumulator, FP16 or BF16 operands, both MN-major
template <class T>
__device__ __forceinline__ uint32_t mma_shape(uint32_t m, uint32_t n) {
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | 1u << 15 | 1u << 16 | (n >> 3) << 17 | (m >> 4) << 24;
}

// Every copy has landed when the products that read it are done.  Where those
// were given up, a copy in flight gets far longer than one takes (2 ms) before
// the CTA may leave.
__device__ __forceinline__ void settle() {
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitClocks / 1000) {}
}

// Few tiles: one 128 x 128 tile per CTA, the tokens split over the CTAs of a
// cluster, and each CTA's run of them over up to 4 accumulators, so that no
// accumulator sums more than it must.  The partial tiles meet in shared memory.
template <class T, int KIND>
__global__ void __launch_bounds__(kThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap map, const Args a) {
    using S = Few;
    constexpr int kStages = S::kStages;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[kStages], empty[kStages], acc_full, drain;
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up_s;
    volatile int* gave_up = &gave_up_s;

    const uint32_t stages = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t parts, part;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
    const uint32_t it0 = part_of(a.iters, part, parts), it1 = part_of(a.iters, part + 1, parts);
    const uint32_t tile = blockIdx.x / parts;
    const uint32_t m0 = tile / a.tiles_n * kBM, n0 = tile % a.tiles_n * S::kBN;

    if (threadIdx.x == 0) {
        gave_up_s = 0;
        for (int s = 0; s < kStages; ++s) {
            bar_init(smem_u32(full + s), kTeam + 1);
            bar_init(smem_u32(empty + s), 1);
        }
        bar_init(smem_u32(&acc_full), 1);
        bar_init(smem_u32(&drain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_at)),
                     "r"(kFewRuns * S::kBN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_at;
    wait_before();

    if (warp == kTmaWarp) {
        const uint32_t me = elect();
        uint32_t s = 0, phase = 0;
        bool ok = true;
        for (uint32_t it = it0; it < it1; ++it) {
            if (!(ok = warp_wait(smem_u32(empty + s), phase ^ 1u, gave_up))) break;
            const uint32_t dst = stages + s * S::kStage + kABytes, bar = smem_u32(full + s);
            bar_expect(bar, S::kBBytes, me);
#pragma unroll
            for (int j = 0; j < S::kBBytes / kAtom; ++j)
                tma_load<false>(dst + j * kAtom, &map, (int)n0 + 64 * j, (int)(it * kBK), bar, me);
            if (++s == kStages) s = 0, phase ^= 1u;
        }
        if (!ok) settle();
    } else if (warp == kMmaWarp) {
        const uint32_t me = elect(), shape = mma_shape<T>(kBM, S::kBN);
        uint32_t s = 0, phase = 0;
        bool ok = true;
        for (uint32_t c = 0; ok && c < a.chunks; ++c) {
            const uint32_t from = it0 + part_of(it1 - it0, c, a.chunks);
            const uint32_t to = it0 + part_of(it1 - it0, c + 1, a.chunks);
            for (uint32_t it = from; it < to; ++it) {
                if (!(ok = warp_wait(smem_u32(full + s), phase, gave_up))) break;
                fence_after();
                const uint64_t x = operand(stages + s * S::kStage), y = x + kABytes / 16;
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k)   // 16 tokens: two groups of 8
                    mma_f16<false>(tmem + c * S::kBN, x + k * (2048 / 16), y + k * (2048 / 16), shape,
                                   it > from || k > 0, me);
                mma_commit<false>(smem_u32(empty + s), me);
                if (++s == kStages) s = 0, phase ^= 1u;
            }
        }
        if (ok) mma_commit<false>(smem_u32(&acc_full), me);
        // no product is in flight when the accumulators are given back
        mma_commit<false>(smem_u32(&drain), me);
        bar_drain(smem_u32(&drain), 0);
    } else if (warp >= kEpiWarps) {
        fill_stages<T, KIND, S::kStage, kStages>(a, it0, it1, m0, stages, empty, full, gave_up);
    } else {
        const bool ok = warp_wait<kSleep>(smem_u32(&acc_full), 0, gave_up);
        fence_after();
        const uint32_t row = warp * 32 + lane;
#pragma unroll 1
        for (int c = 0; c < S::kBN; c += 32) {
            float v[32];
            const uint32_t from = tmem + ((uint32_t)(warp * 32) << 16) + c;
            tmem_ld32(from, reinterpret_cast<uint32_t*>(v));
            for (uint32_t k = 1; k < a.chunks; ++k) {
                float more[32];
                tmem_ld32(from + k * S::kBN, reinterpret_cast<uint32_t*>(more));
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], more[j]);
            }
            if (!ok) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7FC00000u);
            }
            // the stages are idle: every product of this CTA is done
            const uint32_t at = stages + (row * S::kRow + c) * 4;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + j * 4),
                             "f"(v[j]), "f"(v[j + 1]), "f"(v[j + 2]), "f"(v[j + 3])
                             : "memory");
        }
        fence_before();
    }
    __syncwarp();
    cluster_sync();
    // this CTA's share of the tile's rows, four columns per thread, the partial
    // tiles added in rank order
    const uint32_t rows = kBM / parts;
    int lost = 0;   // a partial tile of a CTA that gave up is not to be trusted
    for (uint32_t p = 0; p < parts; ++p) lost |= peer_flag(smem_u32(&gave_up_s), p);
    for (uint32_t i = threadIdx.x; i < rows * (S::kBN / 4); i += kThreads) {
        const uint32_t row = part * rows + i / (S::kBN / 4), col = i % (S::kBN / 4) * 4;
        const uint32_t at = stages + (row * S::kRow + col) * 4;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t p = 0; p < parts; ++p) {
            const float4 q = peer_ld(at, p);
            v[0] = __fadd_rn(v[0], q.x);
            v[1] = __fadd_rn(v[1], q.y);
            v[2] = __fadd_rn(v[2], q.z);
            v[3] = __fadd_rn(v[3], q.w);
        }
        if (lost) v[0] = v[1] = v[2] = v[3] = __uint_as_float(0x7FC00000u);
        out_row4(a.out, a.m, a.n, m0 + row, n0 + col, v, a.accumulate);
    }
    cluster_sync();   // nobody leaves while its tile is read
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(kFewRuns * S::kBN));
    }
}

// Many tiles: pairs of CTAs walk over tiles of 256 x 256 of X (turned into
// 16-bit operands by a pass before) and dY.  Each CTA brings its own 128 columns
// of X and half of dY's; the first one's MMA warp issues products that read
// both.  Per CTA and step that is 32 KB written to and 32 KB read from shared
// memory under 512 clocks of products, where a CTA alone (128 x 256) would move
// 96 KB and be bound by it.
__device__ __forceinline__ void pair_tile(const Args& a, uint32_t t, uint32_t& m, uint32_t& n) {
    // bands of 8 row tiles, so that the tiles at work at one time share both
    // their columns of X and of dY in L2
    const uint32_t band = t / (8 * a.tiles_n), at = t - band * 8 * a.tiles_n;
    const uint32_t high = min(8u, a.tiles_m - band * 8);
    n = at / high;
    m = band * 8 + (at - n * high);
}

// RUNS: several runs of an item's tokens, whose FP32 sums the epilogue adds, and writes
// as FP32 (the partial sums too) or as the output's 16-bit type: two kernels, since all
// three types in one spilled twice as many registers.
enum Runs { kOneRun, kRunsTo32, kRunsTo16 };
template <class T, Runs RUNS>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dy,
                const Args a) {
    using S = Pair;
    constexpr int kStages = S::kStages;
    extern __shared__ uint8_t raw[];
    // full, acc_empty, drain: of the first CTA; the others of each
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up_s;
    volatile int* gave_up = &gave_up_s;

    const uint32_t stages = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    // Items: a tile and a run of the tokens; one run's tiles follow each other, so
    // that the items at work share their rows of X and dY.
    const uint32_t items = a.tiles * a.splits, pairs = gridDim.x / 2;
    auto item = [&](uint32_t i, uint32_t& m, uint32_t& n, uint32_t& it0, uint32_t& it1) {
        const uint32_t run = i / a.tiles;
        pair_tile(a, i - run * a.tiles, m, n);
        it0 = part_of(a.iters, run, a.splits);
        it1 = part_of(a.iters, run + 1, a.splits);
        return run;
    };

    if (threadIdx.x == 0) {
        gave_up_s = 0;
        for (int s = 0; s < kStages; ++s) {
            bar_init(smem_u32(full + s), 1);
            bar_init(smem_u32(empty + s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(smem_u32(acc_full + b), 1);
            bar_init(smem_u32(acc_empty + b), 2 * kPairEpiWarps);
        }
        bar_init(smem_u32(&drain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kPairEpiWarps) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_at)),
                     "r"(2 * S::kBN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    cluster_sync();   // both CTAs' barriers are there before either is used
    fence_after();
    const uint32_t tmem = tmem_at;
    wait_before();

    if (warp == kPairEpiWarps + 1) {
        const uint32_t me = elect();
        uint32_t s = 0, phase = 0;
        bool ok = true;
        for (uint32_t i = blockIdx.x / 2; ok && i < items; i += pairs) {
            uint32_t m, n, it0, it1;
            item(i, m, n, it0, it1);
            const int m0 = (int)(m * 2 * kBM + rank * kBM);
            const int n0 = (int)(n * S::kBN + rank * (S::kBN / 2));
            for (uint32_t it = it0; it < it1; ++it) {
                if (!(ok = warp_wait(smem_u32(empty + s), phase ^ 1u, gave_up))) break;
                const uint32_t dst = stages + s * S::kStage;
                // both CTAs' copies complete on the first one's barrier
                bar_expect(smem_u32(full + s), 2 * S::kStage, me & (rank ^ 1u));
                const uint32_t bar = bar_of(smem_u32(full + s), 0);
#pragma unroll
                for (int j = 0; j < kABytes / kAtom; ++j)
                    tma_load<true>(dst + j * kAtom, &map_x, m0 + 64 * j, (int)(it * kBK), bar, me);
#pragma unroll
                for (int j = 0; j < S::kBBytes / kAtom; ++j)
                    tma_load<true>(dst + kABytes + j * kAtom, &map_dy, n0 + 64 * j, (int)(it * kBK),
                                   bar, me);
                if (++s == kStages) s = 0, phase ^= 1u;
            }
        }
        if (!ok) settle();
    } else if (warp == kPairEpiWarps) {
        if (rank == 0) {
            const uint32_t me = elect(), shape = mma_shape<T>(2 * kBM, S::kBN);
            uint32_t s = 0, phase = 0, buf = 0, bphase = 0;
            bool ok = true;
            for (uint32_t i = blockIdx.x / 2; ok && i < items; i += pairs) {
                uint32_t m, n, it0, it1;
                item(i, m, n, it0, it1);
                for (uint32_t c = 0; ok && c < a.chunks; ++c) {
                    if (!(ok = warp_wait(smem_u32(acc_empty + buf), bphase ^ 1u, gave_up))) break;
                    fence_after();
                    const uint32_t from = it0 + part_of(it1 - it0, c, a.chunks);
                    const uint32_t to = it0 + part_of(it1 - it0, c + 1, a.chunks);
                    for (uint32_t it = from; it < to; ++it) {
                        if (!(ok = warp_wait(smem_u32(full + s), phase, gave_up))) break;
                        fence_after();
                        const uint64_t x = operand(stages + s * S::kStage), y = x + kABytes / 16;
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k)   // 16 tokens: two groups of 8
                            mma_f16<true>(tmem + buf * S::kBN, x + k * (2048 / 16),
                                          y + k * (2048 / 16), shape, it > from || k > 0, me);
                        mma_commit<true>(smem_u32(empty + s), me);
                        if (++s == kStages) s = 0, phase ^= 1u;
                    }
                    if (!ok) break;
                    mma_commit<true>(smem_u32(acc_full + buf), me);
                    if (++buf == 2) buf = 0, bphase ^= 1u;
                }
            }
            // no product is in flight when the accumulators are given back
            mma_commit<true>(smem_u32(&drain), me);
            bar_drain(smem_u32(&drain), 0);
        }
    } else {
        // four warps to each quarter of the rows, a quarter of the columns each
        constexpr int kCols = S::kBN * 4 / kPairEpiWarps;
        const uint32_t quarter = warp % 4, c0 = warp / 4 * kCols;
        float4* staged = reinterpret_cast<float4*>(raw + (stages - smem_u32(raw)) + kStages * S::kStage) +
                         warp * 128;
        Ring<2> acc;
        auto wait = [&] { return warp_wait<kSleep>(smem_u32(acc_full + acc.at), acc.parity, gave_up); };
        // where an item's sums go: its run of tokens, or the output
        auto where = [&](uint32_t run) {
            return a.partial ? Out{a.partial + (uint64_t)run * a.m * a.n_pad, a.n_pad, 1, 0, 1} : a.out;
        };
        const bool accumulate = a.accumulate && !a.partial;
        auto tile = [&](uint32_t i) {
            uint32_t m, n, it0, it1;
            const uint32_t run = item(i, m, n, it0, it1);
            const uint32_t row0 = m * (2 * kBM) + rank * kBM + quarter * 32;
            const Out out = where(run);
            // a lane's 16 columns of one row, among the warp's 32 rows
            auto stage = [&](const float* v) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    staged[lane * 4 + (j ^ (lane >> 1 & 3))] =
                        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                __syncwarp();
            };
            // what is staged, as the columns from c on
            auto put = [&](uint32_t c) {
                const uint32_t col0 = n * S::kBN + c;
                if (RUNS == kRunsTo32 || (RUNS == kOneRun && out.f32))
                    out_block(static_cast<float*>(out.p), out, a.m, a.n, row0, col0, staged, lane, accumulate);
                else if (out.bf16)
                    out_block(static_cast<__nv_bfloat16*>(out.p), out, a.m, a.n, row0, col0, staged, lane,
                              accumulate);
                else
                    out_block(static_cast<__half*>(out.p), out, a.m, a.n, row0, col0, staged, lane, accumulate);
            };
            auto next = [&] {
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_at(bar_of(smem_u32(acc_empty + acc.at), 0));
                acc.next();
            };
            if constexpr (RUNS == kOneRun) {
                if (!wait()) return false;
                fence_after();
#pragma unroll 1
                for (uint32_t c = c0; c < c0 + kCols; c += 16) {
                    float v[16];
                    tmem_ld16(tmem + acc.at * S::kBN + (quarter * 32 << 16) + c,
                              reinterpret_cast<uint32_t*>(v));
                    stage(v);
                    put(c);
                }
                next();
                return true;
            } else {
                // the runs' sums are added in registers
                float sum[kCols / 16][16] = {};
#pragma unroll 1
                for (uint32_t k = 0; k < a.chunks; ++k) {
                    if (!wait()) return false;
                    fence_after();
#pragma unroll
                    for (int c = 0; c < kCols / 16; ++c) {
                        float v[16];
                        tmem_ld16(tmem + acc.at * S::kBN + (quarter * 32 << 16) + c0 + c * 16,
                                  reinterpret_cast<uint32_t*>(v));
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[c][j] = __fadd_rn(sum[c][j], v[j]);
                    }
                    next();
                }
                // unrolled, four copies of the output's code spilled the sums
#pragma unroll 1
                for (int k = 0; k < kCols / 16; ++k) {
#pragma unroll
                    for (int c = 0; c < kCols / 16; ++c)
                        if (c == k) stage(sum[c]);
                    put(c0 + k * 16);
                }
                return true;
            }
        };
        // NaN for the warp's part of a tile
        auto lost = [&](uint32_t i) {
            uint32_t m, n, it0, it1;
            const uint32_t run = item(i, m, n, it0, it1);
            const Out out = where(run);
            const uint32_t row = m * (2 * kBM) + rank * kBM + quarter * 32 + lane, col = n * S::kBN + c0;
            for (uint32_t c = col; row < a.m && c < min(col + kCols, a.n); ++c)
                out_put(out, (uint64_t)row * out.ld + c, __uint_as_float(0x7FC00000u));
        };
        until_lost(blockIdx.x / 2, items, pairs, tile, lost);
    }
    __syncwarp();
    fence_before();
    cluster_sync();   // no product or barrier of the pair is used after this
    if (warp == kPairEpiWarps) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(2 * S::kBN));
    }
    cluster_sync();
}

// the runs' partial sums, added in order: four columns per thread
__global__ void __launch_bounds__(256) runs_kernel(const Args a) {
    wait_before();
    const uint32_t per = a.n_pad / 4;
    const uint64_t total = (uint64_t)a.m * per, run = (uint64_t)a.m * a.n_pad;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(i / per), col = (uint32_t)(i - (uint64_t)row * per) * 4;
        const float* p = a.partial + (uint64_t)row * a.n_pad + col;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t k = 0; k < a.splits; ++k) {
            const float4 q = __ldcs(reinterpret_cast<const float4*>(p + k * run));
            v[0] = __fadd_rn(v[0], q.x);
            v[1] = __fadd_rn(v[1], q.y);
            v[2] = __fadd_rn(v[2], q.z);
            v[3] = __fadd_rn(v[3], q.w);
        }
        out_row4(a.out, a.m, a.n, row, col, v, a.accumulate);
    }
}

// dW of no tokens
__global__ void __launch_bounds__(256) zero_kernel(const Args a) {
    const uint64_t total = (uint64_t)a.m * a.n;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * 256)
        out_put(a.out, i / a.n * a.out.ld + i % a.n, 0.0f);
}

using EncodeFn = decltype(&cuTensorMapEncodeTiled);
EncodeFn encode_fn() {
    static std::atomic<void*> fn{nullptr};
    void* p = fn.load();
    if (!p) {
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return nullptr;
        fn.store(p);
    }
    return reinterpret_cast<EncodeFn>(p);
}

bool tma_rows(const void* p, uint64_t ld, uint64_t cols) {
    return aligned16(p) && ld % 8 == 0 && ld >= cols;
}
uint64_t realigned(uint64_t cols) { return (cols + 7) / 8 * 8; }

// raises a kernel's shared-memory limit, once per device
int set_smem(const void* kernel, int bytes, std::atomic<uint64_t>& ready) {
    if (bytes <= 48 * 1024) return ARK_OK;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ARK_E_CUDA;
    if (dev < 64 && (ready.load() >> dev & 1)) return ARK_OK;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        return ARK_E_CUDA;
    if (dev < 64) ready.fetch_or(1ull << dev);
    return ARK_OK;
}

template <class... P, class... A>
int launch(void (*k)(P...), uint32_t grid, uint32_t threads, int smem, uint32_t cluster,
           std::atomic<uint64_t>& ready, cudaStream_t s, const A&... args) {
    const int rc = set_smem(reinterpret_cast<const void*>(k), smem, ready);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    // blocks may start while the kernel before ends; they wait for its results
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k, args...) == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND>
int launch_few(const CUtensorMap& map, const Args& a, uint32_t parts, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};
    return launch(few_kernel<T, KIND>, a.tiles * parts, kThreads, Few::kSmem, parts, ready, s, map, a);
}
template <class T>
int launch_pair(const CUtensorMap& x, const CUtensorMap& dy, const Args& a, cudaStream_t s) {
    static std::atomic<uint64_t> ready[3];
    const uint32_t most = (uint32_t)sm_count() / 2, items = a.tiles * a.splits;
    const uint32_t pairs = items < most ? items : most;
    auto run = [&](auto kernel, Runs r) {
        return launch(kernel, pairs * 2, kPairThreads, Pair::kSmem, 2, ready[r], s, x, dy, a);
    };
    if (a.chunks == 1) return run(pair_kernel<T, kOneRun>, kOneRun);
    if (a.partial || a.out.f32) return run(pair_kernel<T, kRunsTo32>, kRunsTo32);
    return run(pair_kernel<T, kRunsTo16>, kRunsTo16);
}

// [rows, cols] of 16-bit elements, ld apart, in boxes of 64 columns by 64 rows
int encode(CUtensorMap* map, int32_t type, const void* p, uint64_t rows, uint64_t cols, uint64_t ld) {
    const EncodeFn f = encode_fn();
    if (!f) return ARK_E_CUDA;
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
    const cuuint32_t box[2] = {64, kBK}, ones[2] = {1, 1};
    return f(map,
             type == ARK_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
             2, const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? ARK_OK
               : ARK_E_CUDA;
}

// Clusters of `parts` CTAs of few_kernel that the device holds at once (a GPC's
// SMs do not divide evenly), looked up once per device.
uint32_t few_fit(uint32_t parts) {
    static std::atomic<uint32_t> known[64][4];
    int dev = 0;
    cudaGetDevice(&dev);
    const int at = parts == 1 ? 0 : parts == 2 ? 1 : parts == 4 ? 2 : 3;
    if (dev >= 0 && dev < 64)
        if (const uint32_t n = known[dev][at].load()) return n;
    auto k = few_kernel<__half, kE4M3>;
    cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Few::kSmem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Few::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = sm_count() / (int)parts / 2 + 1;
    }
    if (dev >= 0 && dev < 64) known[dev][at].store((uint32_t)n);
    return (uint32_t)n;
}

// How a gradient is computed, by what each way was measured to take (ns):
//   few_kernel   every wave of CTAs 6500 + 370 for each 64 tokens;
//   pair_kernel  unpack 3000 + its bytes at 5 TB/s; every wave 1500 + 330 for
//                each 64 tokens, 5000 once; split tokens: 3000 + the FP32
//                partial sums written and read at 8 TB/s.
// 512 tokens, 768 x 768: 8.5 us in 72 CTAs of clusters of 2, 13.8 in clusters of
// 4 (144 CTAs, which do not all fit); 8192 tokens: few 30.7, pairs in 8 runs
// 24.3; 8192, 4096 x 4096: pairs 210, few above 600.
struct Way {
    bool pairs;
    uint32_t parts;    // few: CTAs of a cluster
    uint32_t splits;   // pairs: runs of tokens
    uint64_t x_bytes, partial_bytes;
};
Way way_of(uint64_t tokens, uint64_t m, uint64_t n) {
    const uint64_t iters = (tokens + kBK - 1) / kBK, sms = (uint64_t)sm_count();
    const uint64_t few = (m + 127) / 128 * ((n + 127) / 128);
    const uint64_t tiles = (m + 255) / 256 * ((n + 255) / 256);
    auto ceil_div = [](uint64_t a, uint64_t b) { return (a + b - 1) / b; };
    Way w = {false, 1, 1, 0, 0};
    uint64_t best = ~0ull;
    for (uint32_t p = 1; p <= 8 && p <= iters; p *= 2) {
        if (ceil_div(iters, p) > kFewRuns * kFewRun) continue;   // its accumulators take no more
        const uint64_t t = ceil_div(few, few_fit(p)) * (6500 + 370 * ceil_div(iters, p));
        if (t < best) best = t, w.parts = p;
    }
    const uint64_t x_bytes = tokens * act8_pitch(m) * 2, run = m * ((n + 3) / 4 * 4) * 4;
    for (uint32_t r = 1; r <= 16 && (r == 1 || r * 8 <= iters); ++r) {
        const uint64_t waves = ceil_div(tiles * r, sms / 2);
        const uint64_t t = 8000 + x_bytes * 3 / 2 / 5000 + waves * (1500 + 330 * ceil_div(iters, r)) +
                           (r > 1 ? 3000 + 2 * r * run / 8000 : 0);
        if (t < best) best = t, w.pairs = true, w.splits = r;
    }
    if (w.pairs) {
        w.x_bytes = x_bytes;
        w.partial_bytes = w.splits > 1 ? w.splits * run : 0;
    }
    return w;
}
// the workspace's last part: dY realigned
uint64_t ws_dy(uint64_t tokens, const void* dy, uint64_t lddy, uint64_t n) {
    return tma_rows(dy, lddy, n) ? 0 : tokens * realigned(n) * 2;
}

Out out_of(void* dw, int32_t type, uint64_t ld) {
    return Out{dw, ld, type == ARK_TYPE_F32, type == ARK_TYPE_BF16,
               aligned16(dw) && ld * type_size(type) % 16 == 0};
}
// a.partial's runs into a.out
int add_runs(const Args& a, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};
    const uint64_t blocks = ((uint64_t)a.m * a.n_pad / 4 + 255) / 256, most = (uint64_t)sm_count() * 8;
    return launch(runs_kernel, (uint32_t)(blocks < most ? blocks : most), 256, 0, 1, ready, s, a);
}

uint64_t need_of(const Way& w, const ark_act8* x, const void* dy, uint64_t lddy, uint64_t n) {
    return w.x_bytes + w.partial_bytes + ws_dy(x->rows, dy, lddy, n);
}

// The gradient with operands of dY's type; arguments are checked.
int product(const Way& w, const ark_act8* x, const void* dy, int32_t dy_type, uint64_t lddy,
            uint64_t n_out, void* dw, int32_t dw_type, uint64_t lddw, int32_t accumulate, uint8_t* ws,
            cudaStream_t s) {
    Args a = {};
    a.x = x->data;
    a.scale = x->scale;
    a.pitch = act8_pitch(x->cols);
    a.spitch = a.pitch / kActBlock;
    a.tokens = (uint32_t)x->rows;
    a.m = (uint32_t)x->cols;
    a.n = (uint32_t)n_out;
    a.iters = (a.tokens + kBK - 1) / kBK;
    a.out = out_of(dw, dw_type, lddw);
    a.accumulate = accumulate != 0;
    if (x->rows == 0) {
        if (accumulate) return ARK_OK;
        const uint64_t blocks = ((uint64_t)a.m * a.n + 255) / 256;
        zero_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(a);
        return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
    }

    uint64_t ld = lddy;
    if (ws_dy(x->rows, dy, lddy, n_out)) {
        ld = realigned(n_out);
        void* to = ws + w.x_bytes + w.partial_bytes;
        if (const int rc2 = realign_rows(dy, lddy, x->rows, a.n, to, ld, s)) return rc2;
        dy = to;
    }
    CUtensorMap map;
    int failed = encode(&map, dy_type, dy, x->rows, n_out, ld);
    if (failed) return failed;

    if (w.pairs) {
        a.tiles_m = (a.m + 255) / 256;
        a.tiles_n = (a.n + 255) / 256;
        a.tiles = a.tiles_m * a.tiles_n;
        a.splits = w.splits;
        a.partial = w.partial_bytes ? reinterpret_cast<float*>(ws + w.x_bytes) : nullptr;
        a.n_pad = (a.n + 3) / 4 * 4;
        const uint32_t run = (a.iters + a.splits - 1) / a.splits;
        const uint32_t most = a.out.f32 ? kRun32 : a.out.bf16 ? kRunBF16 : kRunF16;
        a.chunks = (run + most - 1) / most;
        failed = act8_operands(x, ws, dy_type, a.pitch, s);
        if (failed) return failed;
        CUtensorMap map_x;
        failed = encode(&map_x, dy_type, ws, x->rows, x->cols, a.pitch);
        if (failed) return failed;
        failed = dy_type == ARK_TYPE_F16 ? launch_pair<__half>(map_x, map, a, s)
                                     : launch_pair<__nv_bfloat16>(map_x, map, a, s);
        if (failed || !a.partial) return failed;
        return add_runs(a, s);
    }
    a.tiles_m = (a.m + kBM - 1) / kBM;
    a.tiles_n = (a.n + Few::kBN - 1) / Few::kBN;
    a.tiles = a.tiles_m * a.tiles_n;
    const uint32_t parts = w.parts;
    a.chunks = a.iters / parts / 16;
    a.chunks = a.chunks < 1 ? 1 : a.chunks > kFewRuns ? kFewRuns : a.chunks;   // of at most kFewRun steps
    if (dy_type == ARK_TYPE_F16)
        return x->kind == kE4M3 ? launch_few<__half, kE4M3>(map, a, parts, s)
                                : launch_few<__half, kInt8>(map, a, parts, s);
    return x->kind == kE4M3 ? launch_few<__nv_bfloat16, kE4M3>(map, a, parts, s)
                            : launch_few<__nv_bfloat16, kInt8>(map, a, parts, s);
}

// dY of FP16 as the sum of two BF16 numbers (8 bits and the 3 that are left; an infinity
// or a NaN stays in the first): 8 columns per thread.
__global__ void __launch_bounds__(256) halves_kernel(const __half* __restrict__ dy, uint64_t lddy,
                                                     uint64_t rows, uint32_t cols, uint32_t per_row,
                                                     __nv_bfloat16* __restrict__ hi,
                                                     __nv_bfloat16* __restrict__ lo, uint64_t ld) {
    const uint64_t total = rows * per_row;
    const bool vec = aligned16(dy) && lddy % 8 == 0;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / per_row;
        const uint32_t col = (uint32_t)(i - row * per_row) * 8;
        float v[8], h[8];
        load8(dy + row * lddy + col, (int)(cols - col), vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[j] = __bfloat162float(__float2bfloat16_rn(v[j]));
            v[j] = isfinite(h[j]) ? __fsub_rn(v[j], h[j]) : 0.0f;
        }
        store_vec<8>(hi + row * ld + col, h);
        store_vec<8>(lo + row * ld + col, v);
    }
}

// Workspace of wide(): both halves of dY, the FP32 gradient, then that of a product.
struct Wide {
    uint64_t ld, ldw, half, sums, inner;   // elements, elements, bytes
    uint64_t bytes() const { return 2 * half + sums + inner; }
};
Wide wide_of(const Way& way, const ark_act8* x, uint64_t n) {
    Wide w;
    w.ld = realigned(n);
    w.ldw = (n + 3) / 4 * 4;
    w.half = x->rows * w.ld * 2;
    w.sums = x->cols * w.ldw * 4;
    w.inner = need_of(way, x, nullptr, w.ld, n);
    return w;
}
// FP16 dY with a checkpoint that FP16 may not hold
int wide(const Way& way, const ark_act8* x, const void* dy, uint64_t lddy, uint64_t n, void* dw,
         int32_t dw_type, uint64_t lddw, int32_t accumulate, uint8_t* ws, cudaStream_t s) {
    const Wide w = wide_of(way, x, n);
    __nv_bfloat16* hi = reinterpret_cast<__nv_bfloat16*>(ws);
    __nv_bfloat16* lo = reinterpret_cast<__nv_bfloat16*>(ws + w.half);
    float* sums = reinterpret_cast<float*>(ws + 2 * w.half);
    uint8_t* inner = ws + 2 * w.half + w.sums;
    const uint32_t per = (uint32_t)(w.ld / 8);
    const uint64_t blocks = (x->rows * per + 255) / 256, most = (uint64_t)sm_count() * 8;
    halves_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(
        static_cast<const __half*>(dy), lddy, x->rows, (uint32_t)n, per, hi, lo, w.ld);
    if (cudaGetLastError() != cudaSuccess) return ARK_E_CUDA;
    int rc = product(way, x, lo, ARK_TYPE_BF16, w.ld, n, sums, ARK_TYPE_F32, w.ldw, 0, inner, s);
    if (!rc) rc = product(way, x, hi, ARK_TYPE_BF16, w.ld, n, sums, ARK_TYPE_F32, w.ldw, 1, inner, s);
    if (rc) return rc;
    Args a = {};
    a.m = (uint32_t)x->cols;
    a.n = (uint32_t)n;
    a.n_pad = (uint32_t)w.ldw;
    a.splits = 1;
    a.partial = sums;
    a.out = out_of(dw, dw_type, lddw);
    a.accumulate = accumulate != 0;
    return add_runs(a, s);
}

}  // namespace
}  // namespace ark

using namespace ark;

extern "C" {

uint64_t ark_cuda_weight_grad_workspace(const ark_act8* x, const void* dy, uint64_t lddy,
                                        uint64_t n_out) {
    if (!x || !x->rows || !x->cols || !n_out) return 0;
    const Way w = way_of(x->rows, x->cols, n_out);
    const uint64_t need = need_of(w, x, dy, lddy, n_out);
    if (!x->wide) return need;
    const uint64_t more = wide_of(w, x, n_out).bytes();   // dY may be FP16
    return need > more ? need : more;
}

int ark_cuda_weight_grad(const ark_act8* x, const void* dy, int32_t dy_type, uint64_t lddy,
                         uint64_t n_out, void* dw, int32_t dw_type, uint64_t lddw,
                         int32_t accumulate, void* workspace, uint64_t workspace_bytes,
                         void* cuda_stream) {
    const int rc = act8_check(x);
    if (rc) return rc;
    if (dy_type != ARK_TYPE_F16 && dy_type != ARK_TYPE_BF16) return ARK_E_UNSUPPORTED;
    if (!type_size(dw_type)) return ARK_E_INVALID_ARG;
    if (x->rows >= (1ull << 31) - kBK || n_out >= (1ull << 31) - 256) return ARK_E_INVALID_ARG;
    if (x->cols > 1 && lddw < n_out) return ARK_E_INVALID_ARG;
    if (x->cols == 0 || n_out == 0) return ARK_OK;
    if (!dw || (x->rows && !dy)) return ARK_E_INVALID_ARG;
    if (x->rows > 1 && lddy < n_out && lddy != 0) return ARK_E_INVALID_ARG;
    const uint64_t e = type_size(dw_type);
    if (!aligned_to(dw, e) || !aligned_to(dy, 2)) return ARK_E_MISALIGNED;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);

    const Way w = x->rows ? way_of(x->rows, x->cols, n_out) : Way{};
    const bool in_halves = x->rows && x->wide && dy_type == ARK_TYPE_F16;
    const uint64_t need = in_halves ? wide_of(w, x, n_out).bytes()
                          : x->rows ? need_of(w, x, dy, lddy, n_out)
                                    : 0;
    if (need) {
        if (!workspace || workspace_bytes < need) return ARK_E_INVALID_ARG;
        if (!aligned16(workspace)) return ARK_E_MISALIGNED;
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (in_halves) return wide(w, x, dy, lddy, n_out, dw, dw_type, lddw, accumulate, ws, s);
    return product(w, x, dy, dy_type, lddy, n_out, dw, dw_type, lddw, accumulate, ws, s);
}

}  // extern "C"
