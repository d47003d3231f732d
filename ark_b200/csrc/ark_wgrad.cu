// ark_wgrad.cu -- the weight gradient of a projection from its input's 8-bit
// checkpoint:  dW[i, o] (+)= sum over tokens t of X[t, i] * dY[t, o].
//
// Both operands have the summed dimension (tokens) as their slow one, so both
// go to the tensor cores MN-major: a stage holds 64 tokens as rows of 128
// bytes (64 columns), 8 rows to a 1024-byte swizzle atom.  dY comes in that
// shape by TMA.  X is read as bytes, 16 per thread, turned into FP16 / BF16 in
// registers (exact: at most 8 significant bits times a power of two) and
// stored to the same swizzled shape, so the 16-bit X never exists in HBM.
//
// Warp roles (14 warps): 0-3 epilogue, 4-11 turn bytes into operands, 12 TMA,
// 13 MMA.  One CTA owns a 128 x BN tile; accumulators are FP32 in TMEM.
// With enough tiles the grid is persistent and two accumulators alternate, so
// that the epilogue of a tile runs under the products of the next one.  With
// few tiles the tokens are split over a cluster of up to 8 CTAs whose FP32
// partial tiles are added over distributed shared memory in rank order: one
// launch, no workspace, the same bits every time.
//
// Every wait is bounded.  One that runs out makes its CTA leave with NaN as
// its tile, which the step's finite check turns into a skipped step.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "ark_act8.cuh"

namespace ark {
namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 4, kCvtWarps = 8;
constexpr int kThreads = (kEpiWarps + kCvtWarps + 2) * 32;
constexpr int kTmaWarp = kEpiWarps + kCvtWarps, kMmaWarp = kTmaWarp + 1;
constexpr int kAtom = kBK * 128;              // 64 tokens x 64 columns of 16 bits
constexpr int kABytes = kBM / 64 * kAtom;
constexpr int kAhead = 3;                     // byte tiles in flight per thread
constexpr uint64_t kWaitNs = 2000000000ull;

template <int BN>
struct Shape {
    static constexpr int kBBytes = BN / 64 * kAtom;
    static constexpr int kStage = kABytes + kBBytes;
    static constexpr int kStages = BN == 256 ? 4 : 6;
    static constexpr int kSmem = kStages * kStage + 1024;  // slack to align to 1024
    static constexpr int kRow = BN + 4;                    // FP32 row of a partial tile
    static_assert(kBM * kRow * 4 <= kStages * kStage, "partial tile fits the stages");
};

struct Args {
    const uint8_t* x;
    const uint8_t* scale;
    uint64_t pitch, spitch;   // bytes
    uint32_t tokens, m, n;
    uint32_t iters;           // 64-token steps in all
    uint32_t tiles_n, tiles;
    void* dw;
    uint64_t ldw;
    int dw_f32, dw_bf16, accumulate, vec;
};

// ------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
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
// false once the wait has run out, or another warp's has
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    if (bar_test(bar, parity)) return true;
    const uint64_t t0 = now_ns();
    for (uint32_t i = 1;; ++i) {
        if (bar_test(bar, parity)) return true;
        if ((i & 63u) == 0) {
            if (*gave_up) return false;
            if (now_ns() - t0 > kWaitNs) {
                *gave_up = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Shared-memory operand, MN-major, 128-byte swizzle: 64-column atoms kAtom
// bytes apart, groups of 8 tokens 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(kAtom >> 4) << 16 |
           (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
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
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
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

// ------------------------------------------------------------ bytes to operands
// Two FP32 values to a pair of T, saturating (a NaN stays one).
__device__ __forceinline__ uint32_t pair_of(float a, float b, __half) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pair_of(float a, float b, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <class T, int KIND>
__device__ __forceinline__ uint4 operand8(uint2 w, uint32_t byte) {
    float v[8];
    dequant8<KIND>(w, byte, v);
    return make_uint4(pair_of(v[0], v[1], T()), pair_of(v[2], v[3], T()),
                      pair_of(v[4], v[5], T()), pair_of(v[6], v[7], T()));
}

// ------------------------------------------------------------ output
__device__ __forceinline__ float dw_get(const Args& a, uint64_t i) {
    if (a.dw_f32) return static_cast<const float*>(a.dw)[i];
    if (a.dw_bf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.dw)[i]);
    return __half2float(static_cast<const __half*>(a.dw)[i]);
}
__device__ __forceinline__ void dw_put(const Args& a, uint64_t i, float v) {
    if (a.dw_f32)
        static_cast<float*>(a.dw)[i] = v;
    else if (a.dw_bf16)
        static_cast<__nv_bfloat16*>(a.dw)[i] = __float2bfloat16_rn(v);
    else
        static_cast<__half*>(a.dw)[i] = __float2half_rn(v);
}
// N (4 or 8) sums of one row, rounded once to the gradient's type
template <int N>
__device__ __forceinline__ void dw_row(const Args& a, uint32_t row, uint32_t col, float* v) {
    if (row >= a.m || col >= a.n) return;
    const uint64_t i = (uint64_t)row * a.ldw + col;
    if (a.vec && col + N <= a.n) {
        float old[N];
        if (a.dw_f32) {
            float* p = static_cast<float*>(a.dw) + i;
            if (a.accumulate) {
                load_vec<N>(p, old);
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = __fadd_rn(v[j], old[j]);
            }
            store_vec<N>(p, v);
        } else if (a.dw_bf16) {
            __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.dw) + i;
            if (a.accumulate) {
                load_vec<N>(p, old);
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = __fadd_rn(v[j], old[j]);
            }
            store_vec<N>(p, v);
        } else {
            __half* p = static_cast<__half*>(a.dw) + i;
            if (a.accumulate) {
                load_vec<N>(p, old);
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = __fadd_rn(v[j], old[j]);
            }
            store_vec<N>(p, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (col + j < a.n)
                dw_put(a, i + j, a.accumulate ? __fadd_rn(v[j], dw_get(a, i + j)) : v[j]);
    }
}

// ------------------------------------------------------------ the kernel
template <int BN, class T, int KIND, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap map, const Args a) {
    using S = Shape<BN>;
    constexpr int kStages = S::kStages;
    constexpr int kBufs = SPLIT ? 1 : 2;
    constexpr int kCols = BN * kBufs;   // TMEM columns: 128, 256 or 512
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[3 * kStages + 2 * kBufs + 1];
    __shared__ uint32_t tmem_at;
    __shared__ int gave_up_s;
    volatile int* gave_up = &gave_up_s;

    const uint32_t stages = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto full_a = [&](int s) { return smem_u32(bars + s); };
    auto full_b = [&](int s) { return smem_u32(bars + kStages + s); };
    auto empty = [&](int s) { return smem_u32(bars + 2 * kStages + s); };
    auto acc_full = [&](int b) { return smem_u32(bars + 3 * kStages + b); };
    auto acc_empty = [&](int b) { return smem_u32(bars + 3 * kStages + kBufs + b); };
    const uint32_t drain = smem_u32(bars + 3 * kStages + 2 * kBufs);

    // this CTA's tiles and its steps of each
    uint32_t parts = 1, part = 0;
    if (SPLIT) {
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
    }
    const uint32_t first = blockIdx.x / parts, step = SPLIT ? a.tiles : gridDim.x;
    const uint32_t it0 = (uint32_t)((uint64_t)a.iters * part / parts);
    const uint32_t it1 = (uint32_t)((uint64_t)a.iters * (part + 1) / parts);
    const uint32_t per_tile = it1 - it0;

    if (threadIdx.x == 0) {
        gave_up_s = 0;
        for (int s = 0; s < kStages; ++s) {
            bar_init(full_a(s), kCvtWarps);
            bar_init(full_b(s), 1);
            bar_init(empty(s), 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            bar_init(acc_full(b), 1);
            bar_init(acc_empty(b), kEpiWarps);
        }
        bar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_at)),
                     "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_at;

    if (warp == kTmaWarp) {
        if (lane == 0) {
            uint32_t s = 0, phase = 0, loads = 0;
            bool ok = true;
            for (uint32_t t = first; ok && t < a.tiles; t += step) {
                const int n0 = (int)(t % a.tiles_n) * BN;
                for (uint32_t it = it0; it < it1; ++it) {
                    if (!(ok = bar_wait(empty(s), phase ^ 1u, gave_up))) break;
                    const uint32_t dst = stages + s * S::kStage + kABytes;
                    bar_expect(full_b(s), S::kBBytes);
                    for (int j = 0; j < BN / 64; ++j)
                        tma_load(dst + j * kAtom, &map, n0 + 64 * j, (int)(it * kBK), full_b(s));
                    ++loads;
                    if (++s == kStages) s = 0, phase ^= 1u;
                }
            }
            // the copies in flight land before the CTA may leave
            for (uint32_t i = 0; i < min(loads, (uint32_t)kStages); ++i) {
                const uint32_t l = loads - 1 - i;
                const uint64_t t0 = now_ns();
                while (!bar_test(full_b((int)(l % kStages)), (l / kStages) & 1u))
                    if (now_ns() - t0 > kWaitNs) break;
            }
        }
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            // FP32 accumulator, both operands MN-major
            const uint32_t idesc = 1u << 4 | type << 7 | type << 10 | 1u << 15 | 1u << 16 |
                                   (uint32_t)(BN >> 3) << 17 | (uint32_t)(kBM >> 4) << 24;
            uint32_t s = 0, phase = 0, buf = 0, bphase = 0;
            bool ok = true;
            for (uint32_t t = first; ok && t < a.tiles; t += step) {
                if (!(ok = bar_wait(acc_empty(buf), bphase ^ 1u, gave_up))) break;
                fence_after();
                for (uint32_t it = it0; it < it1; ++it) {
                    ok = bar_wait(full_b(s), phase, gave_up) && bar_wait(full_a(s), phase, gave_up);
                    if (!ok) break;
                    fence_after();
                    const uint32_t at = stages + s * S::kStage;
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k)   // 16 tokens: two groups of 8
                        mma_f16(tmem + buf * BN, operand(at + k * 2048),
                                operand(at + kABytes + k * 2048), idesc, it > it0 || k > 0);
                    mma_commit(empty(s));
                    if (++s == kStages) s = 0, phase ^= 1u;
                }
                if (!ok) break;
                mma_commit(acc_full(buf));
                if (++buf == kBufs) buf = 0, bphase ^= 1u;
            }
            // no product is in flight when the accumulators are given back
            mma_commit(drain);
            const uint64_t t0 = now_ns();
            while (!bar_test(drain, 0))
                if (now_ns() - t0 > kWaitNs) break;
        }
    } else if (warp >= kEpiWarps) {
        // 16 bytes (half a scale block) of two token rows per thread and step
        const int t = threadIdx.x - kEpiWarps * 32;
        const uint32_t row = t >> 3, unit = t & 7;
        const uint32_t atom = unit >> 2, chunk = (unit & 3) * 2;
        uint4 q[kAhead][2];
        uint32_t sc[kAhead][2];
        uint32_t lt = first, lit = it0;   // what is loaded next
        uint64_t lcol = 0;
        auto load = [&](int p) {
            const bool any = lt < a.tiles;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t tok = lit * kBK + row + 32 * h;
                q[p][h] = make_uint4(0u, 0u, 0u, 0u);
                sc[p][h] = 1;
                if (any && tok < a.tokens) {
                    q[p][h] = __ldg(reinterpret_cast<const uint4*>(a.x + tok * a.pitch + lcol + unit * 16));
                    sc[p][h] = __ldg(a.scale + tok * a.spitch + (lcol >> 5) + (unit >> 1));
                }
            }
            if (++lit == it1) {
                lit = it0;
                lt += step;
                lcol = (uint64_t)(lt / a.tiles_n) * kBM;
            }
        };
        lcol = (uint64_t)(lt / a.tiles_n) * kBM;
#pragma unroll
        for (int p = 0; p < kAhead; ++p) load(p);
        uint32_t todo = 0;
        for (uint32_t i = first; i < a.tiles; i += step) todo += per_tile;
        uint32_t s = 0, phase = 0;
        bool ok = true;
        while (ok && todo) {
#pragma unroll
            for (int p = 0; p < kAhead; ++p) {
                if (!ok || !todo) break;
                if (!(ok = bar_wait(empty(s), phase ^ 1u, gave_up))) break;
                const uint32_t at = stages + s * S::kStage + atom * kAtom;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t r = row + 32 * h;
                    const uint4 lo = operand8<T, KIND>(make_uint2(q[p][h].x, q[p][h].y), sc[p][h]);
                    const uint4 hi = operand8<T, KIND>(make_uint2(q[p][h].z, q[p][h].w), sc[p][h]);
                    // the two atoms' threads store their halves in opposite order: 8
                    // neighbouring lanes then cover all 32 banks
                    const uint4 one = atom ? hi : lo, two = atom ? lo : hi;
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
                if (lane == 0) bar_arrive(full_a(s));
                if (++s == kStages) s = 0, phase ^= 1u;
                --todo;
                load(p);
            }
        }
    } else {
        uint32_t buf = 0, bphase = 0;
        for (uint32_t t = first; t < a.tiles; t += step) {
            const bool ok = bar_wait(acc_full(buf), bphase, gave_up);
            __syncwarp();
            fence_after();
            const uint32_t m0 = t / a.tiles_n * kBM, n0 = t % a.tiles_n * BN;
            const uint32_t row = warp * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                uint32_t r[32];
                tmem_ld32(tmem + buf * BN + ((uint32_t)(warp * 32) << 16) + c, r);
                float* v = reinterpret_cast<float*>(r);
                if (!ok) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7FC00000u);
                }
                if (SPLIT) {
                    // the stages are idle: every product of this CTA is done
                    const uint32_t at = stages + (row * S::kRow + c) * 4;
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + j * 4),
                                     "f"(v[j]), "f"(v[j + 1]), "f"(v[j + 2]), "f"(v[j + 3])
                                     : "memory");
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) dw_row<8>(a, m0 + row, n0 + c + j, v + j);
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_empty(buf));
            if (++buf == kBufs) buf = 0, bphase ^= 1u;
        }
    }

    if (SPLIT) {
        __syncwarp();
        cluster_sync();
        // rows part, part + parts, ... of the tile: four columns per thread, the
        // partial tiles added in rank order
        const uint32_t m0 = first / a.tiles_n * kBM, n0 = first % a.tiles_n * BN;
        const uint32_t rows = kBM / parts;
        int lost = 0;   // a partial tile of a CTA that gave up is not to be trusted
        for (uint32_t p = 0; p < parts; ++p) lost |= peer_flag(smem_u32(&gave_up_s), p);
        for (uint32_t i = threadIdx.x; i < rows * (BN / 4); i += kThreads) {
            const uint32_t row = part * rows + i / (BN / 4), col = i % (BN / 4) * 4;
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
            dw_row<4>(a, m0 + row, n0 + col, v);
        }
        cluster_sync();   // nobody leaves while its tile is read
    }
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// dY whose rows TMA cannot address, copied to rows of a multiple of 16 bytes
__global__ void __launch_bounds__(256) realign_kernel(const uint16_t* __restrict__ src, uint64_t ld,
                                                      uint64_t rows, uint32_t cols,
                                                      uint16_t* __restrict__ dst, uint32_t ldd) {
    const uint32_t per = ldd / 2;
    const uint64_t total = rows * per;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * 256) {
        const uint64_t r = i / per;
        const uint32_t c = (uint32_t)(i - r * per) * 2;
        const uint16_t lo = c < cols ? src[r * ld + c] : (uint16_t)0;
        const uint16_t hi = c + 1 < cols ? src[r * ld + c + 1] : (uint16_t)0;
        *reinterpret_cast<uint32_t*>(dst + r * ldd + c) = pack16(lo, hi);
    }
}

// dW of no tokens
__global__ void __launch_bounds__(256) zero_kernel(const Args a) {
    const uint64_t total = (uint64_t)a.m * a.n;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * 256)
        dw_put(a, i / a.n * a.ldw + i % a.n, 0.0f);
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

template <int BN, class T, int KIND, bool SPLIT>
int launch(const CUtensorMap& map, const Args& a, uint32_t parts, cudaStream_t s) {
    auto k = wgrad_kernel<BN, T, KIND, SPLIT>;
    static std::atomic<uint64_t> ready{0};   // devices whose shared-memory limit is raised
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ARK_E_CUDA;
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 Shape<BN>::kSmem) != cudaSuccess)
            return ARK_E_CUDA;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg = {};
    const uint32_t sms = (uint32_t)sm_count();
    cfg.gridDim = dim3(SPLIT ? a.tiles * parts : (a.tiles < sms ? a.tiles : sms));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<BN>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SPLIT ? parts : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, map, a) == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <int BN, bool SPLIT>
int dispatch(const CUtensorMap& map, const Args& a, int32_t type, int32_t kind, uint32_t parts,
             cudaStream_t s) {
    if (type == ARK_TYPE_F16)
        return kind == kE4M3 ? launch<BN, __half, kE4M3, SPLIT>(map, a, parts, s)
                             : launch<BN, __half, kInt8, SPLIT>(map, a, parts, s);
    return kind == kE4M3 ? launch<BN, __nv_bfloat16, kE4M3, SPLIT>(map, a, parts, s)
                         : launch<BN, __nv_bfloat16, kInt8, SPLIT>(map, a, parts, s);
}

}  // namespace
}  // namespace ark

using namespace ark;

extern "C" {

uint64_t ark_cuda_weight_grad_workspace(uint64_t tokens, const void* dy, uint64_t lddy,
                                        uint64_t n_out) {
    return tma_rows(dy, lddy, n_out) ? 0 : tokens * realigned(n_out) * 2;
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

    Args a = {};
    a.x = x->data;
    a.scale = x->scale;
    a.pitch = act8_pitch(x->cols);
    a.spitch = a.pitch / kActBlock;
    a.tokens = (uint32_t)x->rows;
    a.m = (uint32_t)x->cols;
    a.n = (uint32_t)n_out;
    a.iters = (a.tokens + kBK - 1) / kBK;
    a.dw = dw;
    a.ldw = lddw;
    a.dw_f32 = dw_type == ARK_TYPE_F32;
    a.dw_bf16 = dw_type == ARK_TYPE_BF16;
    a.accumulate = accumulate != 0;
    a.vec = aligned16(dw) && lddw * e % 16 == 0;
    if (x->rows == 0) {
        if (accumulate) return ARK_OK;
        const uint64_t blocks = ((uint64_t)a.m * a.n + 255) / 256;
        zero_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(a);
        return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
    }

    uint64_t ld = lddy;
    if (!tma_rows(dy, lddy, n_out)) {
        ld = realigned(n_out);
        if (!workspace || workspace_bytes < x->rows * ld * 2) return ARK_E_INVALID_ARG;
        if (!aligned16(workspace)) return ARK_E_MISALIGNED;
        const uint64_t blocks = (x->rows * ld / 2 + 255) / 256;
        const uint64_t most = (uint64_t)sm_count() * 8;
        realign_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(
            static_cast<const uint16_t*>(dy), lddy, x->rows, a.n, static_cast<uint16_t*>(workspace),
            (uint32_t)ld);
        if (cudaGetLastError() != cudaSuccess) return ARK_E_CUDA;
        dy = workspace;
    }
    EncodeFn encode = encode_fn();
    if (!encode) return ARK_E_CUDA;
    CUtensorMap map;
    const cuuint64_t dims[2] = {n_out, x->rows}, strides[1] = {ld * 2};
    const cuuint32_t box[2] = {64, kBK}, ones[2] = {1, 1};
    if (encode(&map,
               dy_type == ARK_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
               2, const_cast<void*>(dy), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return ARK_E_CUDA;

    const uint32_t sms = (uint32_t)sm_count(), tiles_m = (a.m + kBM - 1) / kBM;
    const uint32_t wide = tiles_m * ((a.n + 255) / 256);
    if (wide >= sms) {
        a.tiles_n = (a.n + 255) / 256;
        a.tiles = wide;
        return dispatch<256, false>(map, a, dy_type, x->kind, 1, s);
    }
    a.tiles_n = (a.n + 127) / 128;
    a.tiles = tiles_m * a.tiles_n;
    uint32_t parts = 1;
    while (parts < 8 && a.tiles * parts * 2 <= sms && parts * 2 <= a.iters) parts *= 2;
    if (parts == 1) return dispatch<128, false>(map, a, dy_type, x->kind, 1, s);
    return dispatch<128, true>(map, a, dy_type, x->kind, parts, s);
}

}  // extern "C"
