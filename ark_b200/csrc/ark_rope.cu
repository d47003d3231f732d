// ark_rope.cu -- rotary positions of queries and keys, alone or in one pass
// with the RMS norm of each head; the backward of both.
//
//   n = x * rsqrt(mean(x^2) + eps) * gain            (norm, over one head's dim)
//   y1 = n1 cos - n2 sin, y2 = n2 cos + n1 sin       (each rotated pair)
//
// Backward: u = the inverse rotation of dy; h = x * r with r the rsqrt;
//   dgain = sum over tokens and heads of u * h,  dx = r * (u gain - h * mean(u gain h)).
//
// Angles.  A plan holds each pair's turns per position as a 64-bit fraction of
// a turn, so position * fraction wraps exactly at whole turns: the angle of a
// position in the millions is as good as that of the first ones, with one
// integer product and no table in memory.
//
// HBM bounds the rotation alone (131072 tokens, 10 heads of 128, BF16: 88 % of a copy's
// rate).  With the norm, registers do: 4 to 6 blocks an SM, a third of its warps and
// less, of which 55 to 57 % of the issue slots come and 38 to 40 % of the HBM's cycles.
//
// A group of lanes (8 for a head of 128 in 16-bit chunks) takes one token and walks over its heads: the token's cosines and
// sines are formed once, in registers, and nothing is shared between groups,
// so no barrier holds loads back.  A lane owns two chunks of VEC elements that
// hold whole pairs (for the half layout one chunk of each half), the same ones
// of every head, so a pair is rotated in one lane and the gains' gradients
// stay with it.  With few tokens the heads of a token are split over groups.
#include <math.h>
#include <string.h>

#include "ark_act8.cuh"

namespace ark {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxDim = ARK_ROPE_MAX_DIM;
constexpr int kBlocksPerSm = 6;
// More blocks spill: 8192 tokens of 40 heads from e4m3 took 64 us with 4, 78 with
// 5, 101 with 6 (32768: 199, 228, 340).
constexpr int kBackPerSm = 4;

struct Heads {
    void* p;
    uint64_t heads, ts, hs;   // element strides of tokens and heads
};

// How a head's elements are dealt to lanes.
struct Deal {
    uint32_t dim, rot, half;       // half: pairs per head
    uint32_t group;                // lanes per head, a power of two
    uint32_t units, rot_units;     // chunk pairs of a head, and those that are rotated
    int interleaved;
};

struct Args {
    ark_rope_plan plan;
    Deal d;
    const void* pos;
    int pos64, inverse;
    uint64_t tokens, seq;
    uint32_t splits;               // groups that share a token's heads
    Heads q, k, oq, ok;            // inputs (x or dy) and outputs
    const void *gq, *gk;
    int gain_type;
    float eps;
    // checkpoints: written by the forward, read by the backward
    uint8_t *q8, *sq, *k8, *sk;
    uint64_t pq, pk;               // pitches in bytes
    int kind;                      // ARK_ACT8_*, or -1: x comes from xq / xk
    Heads xq, xk;
    float* partial;                // backward: [q blocks + k blocks][dim]
    uint32_t q_blocks, q_splits, k_splits;
};

__device__ __forceinline__ float gain_at(const void* g, int type, uint32_t i) {
    if (type == ARK_TYPE_F32) return static_cast<const float*>(g)[i];
    if (type == ARK_TYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
    return __half2float(static_cast<const __half*>(g)[i]);
}

// position of a token; negative: padding
__device__ __forceinline__ int64_t position(const Args& a, uint64_t t) {
    if (!a.pos) return (int64_t)(t % a.seq);
    return a.pos64 ? static_cast<const long long*>(a.pos)[t]
                   : (int64_t) static_cast<const int*>(a.pos)[t];
}

// ------------------------------------------------------------ a lane's part of a head
// A unit is two chunks of VEC elements: VEC pairs of FP32 for the packed
// instructions, the first chunk's in front (VEC = 1: one pair, the two chunks).

// where unit u's chunks start and whether they are there
template <bool FULL>
struct Unit {
    uint32_t o1, o2, at;   // at: first rotated pair
    bool h1, h2, turned;
};
template <>
struct Unit<true> {        // the whole head is rotated, and no lane is without a unit
    uint32_t o1, o2, at;
    static constexpr bool h1 = true, h2 = true, turned = true;
};
template <int VEC, int G>
__device__ __forceinline__ Unit<(G > 0)> unit_of(const Deal& d, uint32_t u) {
    Unit<(G > 0)> r;
    r.at = u * VEC;
    if constexpr (G > 0) {
        r.o1 = d.interleaved ? u * 2 * VEC : u * VEC;
        r.o2 = d.interleaved ? r.o1 + VEC : G * VEC + u * VEC;
    } else {
        r.turned = u < d.rot_units;
        if (r.turned && !d.interleaved) {
            r.o1 = u * VEC;
            r.o2 = d.half + u * VEC;
        } else {
            r.o1 = r.turned ? u * 2 * VEC : d.rot + (u - d.rot_units) * 2 * VEC;
            r.o2 = r.o1 + VEC;
        }
        r.h1 = u < d.units && r.o1 < d.dim;
        r.h2 = u < d.units && r.o2 < d.dim;
    }
    return r;
}

// the elements as they lie in memory: VEC of each chunk
template <class T, int VEC>
struct Raw {   // 16-bit types
    static constexpr int N = VEC == 1 ? 1 : VEC / 2;
    uint32_t w[2 * N];
    template <class U>
    __device__ __forceinline__ void load(const T* p, const U& u, bool on) {
        if constexpr (VEC == 1) {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
            w[0] = on && u.h1 ? q[u.o1] : 0;
            w[1] = on && u.h2 ? q[u.o2] : 0;
        } else {
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) w[i] = 0;
            if (on && u.h1) part(p + u.o1, w);
            if (on && u.h2) part(p + u.o2, w + N);
        }
    }
    static __device__ __forceinline__ void part(const T* p, uint32_t* w) {
        if constexpr (VEC == 8) {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
        } else if constexpr (VEC == 4) {
            const uint2 q = *reinterpret_cast<const uint2*>(p);
            w[0] = q.x, w[1] = q.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ void get(uint64_t* v) const {
        if constexpr (VEC == 1) {
            float a, b, none;
            widen2(w[0], a, none, T());
            widen2(w[1], b, none, T());
            v[0] = pair(a, b);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float a, b;
                widen2(w[i], a, b, T());
                v[i] = pair(a, b);
            }
        }
    }
    template <class U>
    static __device__ __forceinline__ void put(T* p, const U& u, bool on, const uint64_t* v) {
        float a, b;
        if constexpr (VEC == 1) {
            unpair(v[0], a, b);
            if (on && u.h1) p[u.o1] = Elem<T>::from_f(a);
            if (on && u.h2) p[u.o2] = Elem<T>::from_f(b);
        } else {
            uint32_t w[2 * N];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                unpair(v[i], a, b);
                w[i] = narrow2(a, b, T());
            }
            if constexpr (VEC == 8) {
                if (on && u.h1) *reinterpret_cast<uint4*>(p + u.o1) = make_uint4(w[0], w[1], w[2], w[3]);
                if (on && u.h2) *reinterpret_cast<uint4*>(p + u.o2) = make_uint4(w[4], w[5], w[6], w[7]);
            } else if constexpr (VEC == 4) {
                if (on && u.h1) *reinterpret_cast<uint2*>(p + u.o1) = make_uint2(w[0], w[1]);
                if (on && u.h2) *reinterpret_cast<uint2*>(p + u.o2) = make_uint2(w[2], w[3]);
            } else {
                if (on && u.h1) *reinterpret_cast<uint32_t*>(p + u.o1) = w[0];
                if (on && u.h2) *reinterpret_cast<uint32_t*>(p + u.o2) = w[1];
            }
        }
    }
};
template <int VEC>
struct Raw<float, VEC> {
    float f[2 * VEC];
    template <class U>
    __device__ __forceinline__ void load(const float* p, const U& u, bool on) {
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) f[i] = 0.0f;
        if constexpr (VEC <= 2) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (on && u.h1) f[i] = p[u.o1 + i];
                if (on && u.h2) f[VEC + i] = p[u.o2 + i];
            }
        } else {
            if (on && u.h1) load_vec<VEC>(p + u.o1, f);
            if (on && u.h2) load_vec<VEC>(p + u.o2, f + VEC);
        }
    }
    __device__ __forceinline__ void get(uint64_t* v) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = pair(f[2 * i], f[2 * i + 1]);
    }
    template <class U>
    static __device__ __forceinline__ void put(float* p, const U& u, bool on, const uint64_t* v) {
        float f[2 * VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) unpair(v[i], f[2 * i], f[2 * i + 1]);
        if constexpr (VEC <= 2) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (on && u.h1) p[u.o1 + i] = f[i];
                if (on && u.h2) p[u.o2 + i] = f[VEC + i];
            }
        } else {
            if (on && u.h1) store_vec<VEC>(p + u.o1, f);
            if (on && u.h2) store_vec<VEC>(p + u.o2, f + VEC);
        }
    }
};

// FP32 of shared memory (zero where the head ends) as a unit's pairs
template <int VEC, class U>
__device__ __forceinline__ void unit_floats(const float* p, const U& u, uint64_t* v) {
    if constexpr (VEC == 1) {
        v[0] = pair(u.h1 ? p[u.o1] : 0.0f, u.h2 ? p[u.o2] : 0.0f);
    } else if constexpr (VEC == 2) {
        const float2 a = u.h1 ? *reinterpret_cast<const float2*>(p + u.o1) : float2{};
        const float2 b = u.h2 ? *reinterpret_cast<const float2*>(p + u.o2) : float2{};
        v[0] = pair(a.x, a.y), v[1] = pair(b.x, b.y);
    } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; i += 2) {
            const float4 a = u.h1 ? *reinterpret_cast<const float4*>(p + u.o1 + 2 * i) : float4{};
            const float4 b = u.h2 ? *reinterpret_cast<const float4*>(p + u.o2 + 2 * i) : float4{};
            v[i] = pair(a.x, a.y), v[i + 1] = pair(a.z, a.w);
            v[VEC / 2 + i] = pair(b.x, b.y), v[VEC / 2 + i + 1] = pair(b.z, b.w);
        }
    }
}

// cos and sin (times the plan's gain) of a unit's VEC rotated pairs
// T: what the result is rounded to.  FP32 holds 24 of the turn's 32 bits, 2^-25 of a
// half turn, which is nothing beside a 16-bit result's half step; for an FP32 result
// the 8 bits below turn it on by an angle too small for more than its first power.
template <class T, int VEC>
struct Turn {
    float c[VEC], s[VEC];
    __device__ __forceinline__ void set(const Args& a, const uint64_t* turns, int64_t p) {
        constexpr float kHalfTurn = 4.656612873077392578125e-10f;   // 2^-31
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            // the top 32 bits of the turn, signed: [-1/2, 1/2) of a turn
            const int32_t top = (int32_t)(((uint64_t)p * turns[i]) >> 32);
            if constexpr (std::is_same<T, float>::value) {
                sincospif(__fmul_rn((float)(top & ~255), kHalfTurn), &s[i], &c[i]);
                const float on = __fmul_rn((float)(top & 255), 3.14159265f * kHalfTurn);
                const float turned = __fmaf_rn(c[i], on, s[i]);
                c[i] = __fmaf_rn(-s[i], on, c[i]);
                s[i] = turned;
            } else {
                sincospif(__fmul_rn((float)top, kHalfTurn), &s[i], &c[i]);
            }
            c[i] = __fmul_rn(c[i], a.plan.gain);
            s[i] = __fmul_rn(a.inverse ? -s[i] : s[i], a.plan.gain);
        }
    }
    // Rotate a unit's pairs in place.  A layout's products are rounded in one order, whatever
    // the width of a chunk: results do not depend on how rows are aligned.
    __device__ __forceinline__ void operator()(const Deal& d, uint64_t* v) const {
        if (d.interleaved) {   // both of a rotated pair in one register pair
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float x, y;
                unpair(v[i], x, y);
                v[i] = pair(__fmaf_rn(x, c[i], -__fmul_rn(y, s[i])),
                            __fmaf_rn(y, c[i], __fmul_rn(x, s[i])));
            }
        } else if constexpr (VEC == 1) {
            float x, y;
            unpair(v[0], x, y);
            v[0] = pair(__fmaf_rn(y, -s[0], __fmul_rn(x, c[0])), __fmaf_rn(y, c[0], __fmul_rn(x, s[0])));
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                const uint64_t x = v[i], y = v[i + VEC / 2];
                const uint64_t cc = pair(c[2 * i], c[2 * i + 1]), ss = pair(s[2 * i], s[2 * i + 1]);
                v[i] = fma2(y, neg2(ss), mul2(x, cc));
                v[i + VEC / 2] = fma2(y, cc, mul2(x, ss));
            }
        }
    }
};

// G: the group's lanes, 0 where they are not known before the launch
template <int G>
__device__ __forceinline__ float group_sum(float v, uint32_t group) {
    if constexpr (G > 0) {
#pragma unroll
        for (int o = G >> 1; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    } else {
        for (uint32_t o = group >> 1; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    }
    return v;
}

// Checkpoint the two chunks of 8 of a lane.  A scale block is 4 lanes' chunks
// of one half (half layout), or both chunks of 2 lanes (then they adjoin).
template <int KIND, int G, class T, class U>
__device__ __forceinline__ void hold(uint8_t* data, uint8_t* scale, uint64_t col, const U& u, bool on,
                                     const Raw<T, 8>& x) {
    const bool next = u.o2 == u.o1 + 8;
    uint32_t q[4], b1, b2;
    if constexpr (std::is_same<T, float>::value) {
        uint32_t m1 = abs_max<8>(x.f), m2 = abs_max<8>(x.f + 8);
        if (next) m1 = m2 = max(m1, m2);
        m1 = max(m1, __shfl_xor_sync(0xFFFFFFFFu, m1, 1));
        m2 = max(m2, __shfl_xor_sync(0xFFFFFFFFu, m2, 1));
        const uint32_t n1 = __shfl_xor_sync(0xFFFFFFFFu, m1, 2), n2 = __shfl_xor_sync(0xFFFFFFFFu, m2, 2);
        if (!next) m1 = max(m1, n1), m2 = max(m2, n2);
        if (!on || !u.h1) return;
        b1 = scale_byte<KIND>(m1), b2 = scale_byte<KIND>(m2);
        const uint2 a = quant8<KIND>(x.f, b1), b = quant8<KIND>(x.f + 8, b2);
        q[0] = a.x, q[1] = a.y, q[2] = b.x, q[3] = b.y;
    } else {
        // the chunks' maxima as the two halves of a word
        const uint32_t a = pairs_max<4>(x.w), b = pairs_max<4>(x.w + 4);
        uint32_t m = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
        if (next) m = __vmaxu2(m, __byte_perm(m, m, 0x1032));
        m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        const uint32_t n = __shfl_xor_sync(0xFFFFFFFFu, m, 2);
        if (!next) m = __vmaxu2(m, n);
        float f1, f2;
        widen2(m, f1, f2, T());
        b1 = scale_byte<KIND>(__float_as_uint(f1)), b2 = scale_byte<KIND>(__float_as_uint(f2));
        if constexpr (G > 0) {   // the head's 2 or 4 scale bytes as one store
            uint32_t all = b1 << (u.o1 >> 5) * 8 | b2 << (u.o2 >> 5) * 8;
            all |= __shfl_xor_sync(0xFFFFFFFFu, all, 2);
            if (G == 8) all |= __shfl_xor_sync(0xFFFFFFFFu, all, 4);
            if (on && u.o1 == 0) {
                if (G == 8)
                    *reinterpret_cast<uint32_t*>(scale + (col >> 5)) = all;
                else
                    *reinterpret_cast<uint16_t*>(scale + (col >> 5)) = (uint16_t)all;
            }
        }
        if (!on || !u.h1) return;
        quant_words<T, KIND, 4>(x.w, b1, q);
        quant_words<T, KIND, 4>(x.w + 4, b2, q + 2);
    }
    *reinterpret_cast<uint2*>(data + col + u.o1) = make_uint2(q[0], q[1]);
    *reinterpret_cast<uint2*>(data + col + u.o2) = make_uint2(q[2], q[3]);
    if (G == 0 && (u.o1 & 31u) == 0) scale[(col + u.o1) >> 5] = (uint8_t)b1;
    if (G == 0 && (u.o2 & 31u) == 0) scale[(col + u.o2) >> 5] = (uint8_t)b2;
}

// a row's columns behind the last head, up to the pitch
__device__ __forceinline__ void hold_rest(uint8_t* data, uint8_t* scale, uint64_t cols,
                                          uint64_t pitch, uint32_t lane, uint32_t lanes) {
    for (uint64_t c = cols + lane * 32; c < pitch; c += lanes * 32) {
        *reinterpret_cast<uint4*>(data + c) = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(data + c + 16) = make_uint4(0u, 0u, 0u, 0u);
        scale[c >> 5] = 1;
    }
}

// What a group of lanes does at a time: a token, a split of its heads.  The groups
// of a warp take neighbouring tokens and the same split, so that they go through
// queries and keys together; all its lanes take every round, since groups shuffle
// together.
struct Task {
    uint64_t t;
    uint32_t lo, hi;   // heads
    int64_t p;         // position
    bool on, live;
    __device__ __forceinline__ Task(const Args& a, uint32_t group, uint64_t warp, uint32_t heads,
                                    uint32_t splits) {
        const uint64_t block = splits == 1 ? warp : warp / splits;
        const uint32_t split = (uint32_t)(warp - block * splits);
        t = block * (32 / group) + (threadIdx.x & 31) / group;
        on = t < a.tokens;
        if (!on) t = 0;
        const uint32_t per = (heads + splits - 1) / splits;
        lo = on ? min(split * per, heads) : 0;
        hi = on ? min(lo + per, heads) : 0;
        p = on ? position(a, t) : -1;
        live = p >= 0;
    }
};
__device__ __forceinline__ uint64_t warp_tasks(const Args& a, uint32_t splits) {
    const uint32_t in_warp = 32 / a.d.group;
    return (a.tokens + in_warp - 1) / in_warp * splits;
}

// ------------------------------------------------------------ forward
// HOLD: 0 no checkpoint, 1 e4m3, 2 int8.  A padding token's outputs are zero,
// and so is the checkpoint that is made here (one by a launch of its own holds
// what the padding holds; nothing reads either).
// G: lanes of a group where the whole head is rotated and 16 G long, else 0: then
// nothing of a head's shape is known before the launch.
template <class T, int VEC, int NU, int G, bool NORM, int HOLD>
__global__ void __launch_bounds__(kThreads, NU == 1 ? kBlocksPerSm : 4) forward_kernel(const __grid_constant__ Args a) {
    // two heads in flight per lane, where a head is few registers
    constexpr int kHeads = NU == 1 && sizeof(T) == 2 ? 2 : 1;
    __shared__ uint64_t turns[kMaxDim / 2];
    __shared__ __align__(16) float gains[NORM ? 2 * kMaxDim : 4];
    const Deal& d = a.d;
    const uint32_t group = G > 0 ? G : d.group, dim = G > 0 ? 2 * VEC * G : d.dim;
    for (uint32_t i = threadIdx.x; i < d.half; i += kThreads) turns[i] = a.plan.turns[i];
    if (NORM)
        for (uint32_t i = threadIdx.x; i < dim; i += kThreads) {
            gains[i] = gain_at(a.gq, a.gain_type, i);
            gains[kMaxDim + i] = a.k.heads ? gain_at(a.gk, a.gain_type, i) : 0.0f;
        }
    __syncthreads();
    const uint32_t lane = threadIdx.x & (group - 1);
    const uint32_t hq = (uint32_t)a.q.heads, heads = hq + (uint32_t)a.k.heads;
    const float inv_dim = __fdiv_rn(1.0f, (float)dim);
    Unit<(G > 0)> u[NU];
#pragma unroll
    for (int n = 0; n < NU; ++n) u[n] = unit_of<VEC, G>(d, lane + n * group);

    const uint64_t tasks = warp_tasks(a, a.splits), stride = (uint64_t)gridDim.x * (kThreads / 32);
    for (uint64_t w = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); w < tasks; w += stride) {
        const Task k(a, group, w, heads, a.splits);
        Turn<T, VEC> turn[NU];
#pragma unroll
        for (int n = 0; n < NU; ++n)
            if (u[n].turned && u[n].h1) turn[n].set(a, turns + u[n].at, k.p);
        // the queries among the task's heads, then the keys
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
            const uint32_t from = part ? max(k.lo, hq) - hq : min(k.lo, hq);
            const uint32_t to = part ? max(k.hi, hq) - hq : min(k.hi, hq);
            const uint32_t rounds = __reduce_max_sync(0xFFFFFFFFu, to - from);
            if (!rounds) continue;
            const Heads& in = part ? a.k : a.q;
            const Heads& out = part ? a.ok : a.oq;
            const T* x = static_cast<const T*>(in.p) + k.t * in.ts + from * in.hs;
            T* y = static_cast<T*>(out.p) + k.t * out.ts + from * out.hs;
            const uint64_t pitch = part ? a.pk : a.pq;
            uint8_t* data = (part ? a.k8 : a.q8) + k.t * pitch;
            uint8_t* scale = (part ? a.sk : a.sq) + k.t * (pitch >> 5);
            uint64_t col = (uint64_t)from * dim;
            const float* g = gains + (part ? kMaxDim : 0);
            for (uint32_t h = 0; h < rounds; h += kHeads) {
                Raw<T, VEC> raw[kHeads][NU];
#pragma unroll
                for (int j = 0; j < kHeads; ++j)
#pragma unroll
                    for (int n = 0; n < NU; ++n)
                        raw[j][n].load(x + j * in.hs, u[n], k.live && from + h + j < to);
#pragma unroll
                for (int j = 0; j < kHeads; ++j) {
                    const bool here = from + h + j < to;
                    if constexpr (HOLD != 0 && VEC == 8)
                        hold<HOLD - 1, G>(data, scale, col, u[0], here, raw[j][0]);
                    uint64_t v[NU][VEC];
#pragma unroll
                    for (int n = 0; n < NU; ++n) raw[j][n].get(v[n]);
                    if (NORM) {
                        uint64_t ss = 0;
#pragma unroll
                        for (int n = 0; n < NU; ++n)
#pragma unroll
                            for (int i = 0; i < VEC; ++i) ss = fma2(v[n][i], v[n][i], ss);
                        const float all = group_sum<G>(sum2(ss), group);
                        const uint64_t r = twice(rsqrtf(__fmaf_rn(all, inv_dim, a.eps)));
#pragma unroll
                        for (int n = 0; n < NU; ++n) {
                            uint64_t gain[VEC];
                            unit_floats<VEC>(g, u[n], gain);
#pragma unroll
                            for (int i = 0; i < VEC; ++i) v[n][i] = mul2(mul2(v[n][i], r), gain[i]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NU; ++n) {
                        if (u[n].turned) turn[n](d, v[n]);
                        if (!k.live) {
#pragma unroll
                            for (int i = 0; i < VEC; ++i) v[n][i] = 0;
                        }
                        Raw<T, VEC>::put(y, u[n], here, v[n]);
                    }
                    x += in.hs;
                    y += out.hs;
                    col += dim;
                }
            }
        }
        if constexpr (HOLD != 0 && VEC == 8) {
            if (k.on && k.lo == 0) {
                hold_rest(a.q8 + k.t * a.pq, a.sq + k.t * (a.pq >> 5), a.q.heads * dim, a.pq, lane,
                          group);
                if (a.k.heads)
                    hold_rest(a.k8 + k.t * a.pk, a.sk + k.t * (a.pk >> 5), a.k.heads * dim, a.pk, lane,
                              group);
            }
        }
    }
}

// ------------------------------------------------------------ backward
// A unit's stored bytes as they lie in memory, and its two scale bytes.
template <int VEC, int G>
struct Bytes {
    uint32_t w[VEC == 8 ? 4 : 2];
    uint32_t s1, s2;
    static __device__ __forceinline__ void part(const uint8_t* p, uint32_t* w) {
        if constexpr (VEC == 8) {
            const uint2 q = *reinterpret_cast<const uint2*>(p);
            w[0] = q.x, w[1] = q.y;
        } else if constexpr (VEC == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (VEC == 2) {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        } else {
            w[0] = *p;
        }
    }
    template <class U>
    __device__ __forceinline__ void load(const uint8_t* data, const uint8_t* scale, uint64_t col,
                                         const U& u, bool on) {
        constexpr int kHalf = VEC == 8 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < 2 * kHalf; ++i) w[i] = 0;
        s1 = s2 = 127;
        if constexpr (G == 8) {   // the head's four scale bytes are a word
            if (on) {
                const uint32_t all = *reinterpret_cast<const uint32_t*>(scale + (col >> 5));
                s1 = all >> (u.o1 >> 5) * 8 & 255u;
                s2 = all >> (u.o2 >> 5) * 8 & 255u;
            }
        } else {
            if (on && u.h1) s1 = scale[(col + u.o1) >> 5];
            if (on && u.h2) s2 = scale[(col + u.o2) >> 5];
        }
        if (on && u.h1) part(data + col + u.o1, w);
        if (on && u.h2) part(data + col + u.o2, w + kHalf);
    }
    // the values before scaling, and the chunks' scales
    template <int KIND>
    __device__ __forceinline__ void get(uint64_t* v, float& f1, float& f2) const {
        f1 = scale_of(s1), f2 = scale_of(s2);
        float b[4], c[4];
        if constexpr (VEC == 1) {
            bytes4<KIND>(w[0], b);
            bytes4<KIND>(w[1], c);
            v[0] = pair(b[0], c[0]);
        } else if constexpr (VEC == 2) {
            bytes4<KIND>(w[0], b);
            bytes4<KIND>(w[1], c);
            v[0] = pair(b[0], b[1]), v[1] = pair(c[0], c[1]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                bytes4<KIND>(w[i], b);
                v[2 * i] = pair(b[0], b[1]), v[2 * i + 1] = pair(b[2], b[3]);
            }
        }
    }
};
template <class T, int VEC, int G, int SRC>
struct Source {   // x as T
    Raw<T, VEC> r;
    __device__ __forceinline__ void get(uint64_t* v, float& f1, float& f2) const {
        r.get(v);
        f1 = f2 = 1.0f;
    }
};
template <class T, int VEC, int G>
struct Source<T, VEC, G, 1> {
    Bytes<VEC, G> r;
    __device__ __forceinline__ void get(uint64_t* v, float& f1, float& f2) const {
        r.template get<kE4M3>(v, f1, f2);
    }
};
template <class T, int VEC, int G>
struct Source<T, VEC, G, 2> {
    Bytes<VEC, G> r;
    __device__ __forceinline__ void get(uint64_t* v, float& f1, float& f2) const {
        r.template get<kInt8>(v, f1, f2);
    }
};

// The blocks below a.q_blocks take the queries, the others the keys, so that a
// lane's running gradient belongs to one gain.  Each block leaves its sums in
// a.partial; gains_kernel adds them in block order.  The next head's loads are
// issued before a head is worked on.
// SRC: 0 x as T, 1 e4m3, 2 int8.
template <class T, int VEC, int NU, int G, int SRC>
__global__ void __launch_bounds__(kThreads, kBackPerSm)
    backward_kernel(const __grid_constant__ Args a) {
    __shared__ uint64_t turns[kMaxDim / 2];
    __shared__ __align__(16) float gains[kMaxDim];
    extern __shared__ float sums[];   // at the end [groups][dim]
    const Deal& d = a.d;
    const uint32_t group = G > 0 ? G : d.group, dim = G > 0 ? 2 * VEC * G : d.dim;
    const bool is_q = blockIdx.x < a.q_blocks;
    const void* gain = is_q ? a.gq : a.gk;
    for (uint32_t i = threadIdx.x; i < d.half; i += kThreads) turns[i] = a.plan.turns[i];
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) gains[i] = gain_at(gain, a.gain_type, i);
    __syncthreads();
    const uint32_t block = is_q ? blockIdx.x : blockIdx.x - a.q_blocks;
    const uint32_t blocks = is_q ? a.q_blocks : gridDim.x - a.q_blocks;
    const Heads &in = is_q ? a.q : a.k, &out = is_q ? a.oq : a.ok, &src = is_q ? a.xq : a.xk;
    const uint32_t heads = (uint32_t)in.heads, splits = is_q ? a.q_splits : a.k_splits;
    const uint64_t pitch = is_q ? a.pq : a.pk;

    const uint32_t lane = threadIdx.x & (group - 1);
    const float inv_dim = __fdiv_rn(1.0f, (float)dim);
    Unit<(G > 0)> u[NU];
    uint64_t dg[NU][VEC];
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        u[n] = unit_of<VEC, G>(d, lane + n * group);
#pragma unroll
        for (int i = 0; i < VEC; ++i) dg[n][i] = 0;
    }
    const uint64_t tasks = warp_tasks(a, splits), stride = (uint64_t)blocks * (kThreads / 32);
    for (uint64_t w = (uint64_t)block * (kThreads / 32) + (threadIdx.x >> 5); w < tasks; w += stride) {
        const Task k(a, group, w, heads, splits);
        const uint32_t count = k.hi - k.lo, rounds = __reduce_max_sync(0xFFFFFFFFu, count);
        const T* dy = static_cast<const T*>(in.p) + k.t * in.ts + k.lo * in.hs;
        const T* xp = static_cast<const T*>(src.p) + k.t * src.ts + k.lo * src.hs;
        const uint8_t* data = (is_q ? a.q8 : a.k8) + k.t * pitch;
        const uint8_t* scale = (is_q ? a.sq : a.sk) + k.t * (pitch >> 5);
        uint64_t col = (uint64_t)k.lo * dim;
        T* dx = static_cast<T*>(out.p) + k.t * out.ts + k.lo * out.hs;
        Raw<T, VEC> g0[NU];
        Source<T, VEC, G, SRC> x0[NU];
        auto load = [&](uint32_t h) {
            const bool read = k.live && h < count;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                g0[n].load(dy, u[n], read);
                if constexpr (SRC == 0)
                    x0[n].r.load(xp, u[n], read);
                else
                    x0[n].r.load(data, scale, col, u[n], read);
            }
            dy += in.hs;
            if (SRC == 0) xp += src.hs;
            col += dim;
        };
        load(0);
        Turn<T, VEC> turn[NU];
#pragma unroll
        for (int n = 0; n < NU; ++n)
            if (u[n].turned && u[n].h1) turn[n].set(a, turns + u[n].at, k.p);
        for (uint32_t h = 0; h < rounds; ++h) {
            const bool here = h < count, read = here && k.live;
            uint64_t v[NU][VEC], x[NU][VEC];
            float f1[NU], f2[NU];
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                g0[n].get(v[n]);
                x0[n].get(x[n], f1[n], f2[n]);
            }
            load(h + 1);
            // the squares before scaling, then scaled twice: no scale's square is formed
            float own = 0.0f;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                if constexpr (VEC == 1) {
                    float b, c;
                    unpair(mul2(x[n][0], x[n][0]), b, c);
                    own = __fadd_rn(own, __fadd_rn(__fmul_rn(__fmul_rn(b, f1[n]), f1[n]),
                                                   __fmul_rn(__fmul_rn(c, f2[n]), f2[n])));
                } else {
                    uint64_t q1 = 0, q2 = 0;
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        q1 = fma2(x[n][i], x[n][i], q1);
                        q2 = fma2(x[n][VEC / 2 + i], x[n][VEC / 2 + i], q2);
                    }
                    own = __fadd_rn(own, __fadd_rn(__fmul_rn(__fmul_rn(sum2(q1), f1[n]), f1[n]),
                                                   __fmul_rn(__fmul_rn(sum2(q2), f2[n]), f2[n])));
                }
            }
            const float all = group_sum<G>(own, group);
            // nothing of a padding token may reach the sums, not even 0 * rsqrt(0)
            const float r1 = read ? rsqrtf(__fmaf_rn(all, inv_dim, a.eps)) : 0.0f;
            const uint64_t r = twice(r1);
            uint64_t dot2 = 0;
#pragma unroll
            for (int n = 0; n < NU; ++n) {
                if (u[n].turned && read) turn[n](d, v[n]);
                uint64_t g[VEC];
                unit_floats<VEC>(gains, u[n], g);
                const float e1 = __fmul_rn(f1[n], r1), e2 = __fmul_rn(f2[n], r1);
                const uint64_t h1 = VEC == 1 ? pair(e1, e2) : twice(e1), h2 = twice(e2);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    x[n][i] = mul2(x[n][i], i < VEC / 2 || VEC == 1 ? h1 : h2);
                    dg[n][i] = fma2(v[n][i], x[n][i], dg[n][i]);
                    v[n][i] = mul2(v[n][i], g[i]);
                    dot2 = fma2(v[n][i], x[n][i], dot2);
                }
            }
            const uint64_t dot = twice(-__fmul_rn(group_sum<G>(sum2(dot2), group), inv_dim));
#pragma unroll
            for (int n = 0; n < NU; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[n][i] = mul2(fma2(x[n][i], dot, v[n][i]), r);
                Raw<T, VEC>::put(dx, u[n], here, v[n]);
            }
            dx += out.hs;
        }
    }
    // the groups' sums, added in group order
    const uint32_t mine = threadIdx.x / group, groups = kThreads / group;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        float f[2 * VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) unpair(dg[n][i], f[2 * i], f[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (u[n].h1) sums[mine * dim + u[n].o1 + i] = f[i];
            if (u[n].h2) sums[mine * dim + u[n].o2 + i] = f[VEC + i];
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) {
        float s = 0.0f;
        for (uint32_t m = 0; m < groups; ++m) s = __fadd_rn(s, sums[m * dim + i]);
        a.partial[(uint64_t)blockIdx.x * dim + i] = s;
    }
}

// blocks' sums to the gains' gradients: one warp per element, in a fixed order
__global__ void __launch_bounds__(kThreads) gains_kernel(const float* __restrict__ partial,
                                                         uint32_t q_blocks, uint32_t blocks,
                                                         uint32_t dim, void* dgq, void* dgk,
                                                         int type, int accumulate) {
    const uint32_t at = (blockIdx.x * kThreads + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    const bool is_q = at < dim;
    const uint32_t i = is_q ? at : at - dim;
    if (i >= dim) return;
    const uint32_t lo = is_q ? 0 : q_blocks, hi = is_q ? q_blocks : blocks;
    void* out = is_q ? dgq : dgk;
    if (!out) return;   // no such gain; one of no heads gets zero
    float s = 0.0f;
    for (uint32_t b = lo + lane; b < hi; b += 32) s = __fadd_rn(s, partial[(uint64_t)b * dim + i]);
    s = group_sum<32>(s, 32);
    if (lane) return;
    if (accumulate) s = __fadd_rn(s, gain_at(out, type, i));
    if (type == ARK_TYPE_F32)
        static_cast<float*>(out)[i] = s;
    else if (type == ARK_TYPE_BF16)
        static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(s);
    else
        static_cast<__half*>(out)[i] = __float2half_rn(s);
}

// ------------------------------------------------------------ host
Heads heads_of(const ark_heads* h) {
    return h ? Heads{h->data, h->heads, h->token_stride, h->head_stride} : Heads{nullptr, 0, 0, 0};
}

bool heads_ok(const Heads& h, uint64_t tokens, uint64_t dim, uint64_t e, bool written, int* rc) {
    if (h.heads == 0 || tokens == 0) return true;
    if (!h.p || h.heads >= (1u << 16)) {
        *rc = ARK_E_INVALID_ARG;
        return false;
    }
    if (!aligned_to(h.p, e)) {
        *rc = ARK_E_MISALIGNED;
        return false;
    }
    // written heads may not overlap, in either order of tokens and heads
    if (written) {
        const bool inner = (h.heads == 1 || h.hs >= dim) &&
                           (tokens == 1 || h.ts >= (h.heads - 1) * h.hs + dim);
        const bool outer = (tokens == 1 || h.ts >= dim) &&
                           (h.heads == 1 || h.hs >= (tokens - 1) * h.ts + dim);
        if (!inner && !outer) {
            *rc = ARK_E_INVALID_ARG;
            return false;
        }
    }
    return true;
}

// elements that every row of a set of heads starts at a multiple of
bool multiple(const Heads& h, uint64_t e, uint64_t vec) {
    if (h.heads == 0) return true;
    const uint64_t bytes = vec * e > 16 ? 16 : vec * e;
    return aligned_to(h.p, bytes) && h.ts * e % bytes == 0 && h.hs * e % bytes == 0;
}

// The widest chunk that divides the head, its rotated part and every row's start.
int chunk_of(const ark_rope_plan* p, uint64_t dim, uint64_t e, const Heads* h, int n) {
    for (int vec = 8; vec > 1; vec /= 2) {
        const uint64_t rot = p->rotary_dim;
        bool ok = dim % vec == 0 && (p->interleaved ? rot % (2 * vec) == 0 : rot / 2 % vec == 0);
        for (int i = 0; ok && i < n; ++i) ok = multiple(h[i], e, (uint64_t)vec);
        if (ok) return vec;
    }
    return 1;
}

Deal deal_of(const ark_rope_plan* p, uint64_t dim, int vec) {
    Deal d;
    d.dim = (uint32_t)dim;
    d.rot = p->rotary_dim;
    d.half = d.rot / 2;
    d.interleaved = p->interleaved != 0;
    d.rot_units = d.half / vec;
    d.units = d.rot_units + (d.dim - d.rot + 2 * vec - 1) / (2 * vec);
    d.group = 1;
    while (d.group < 32 && d.group < d.units) d.group *= 2;
    return d;
}

int plan_ok(const ark_rope_plan* p, uint64_t dim) {
    if (!p || p->rotary_dim < 2 || p->rotary_dim % 2 || p->interleaved > 1) return ARK_E_INVALID_ARG;
    if (dim > kMaxDim) return ARK_E_UNSUPPORTED;
    return p->rotary_dim <= dim ? ARK_OK : ARK_E_INVALID_ARG;
}

int common_ok(const Args& a, uint64_t e, uint64_t dim, int pos_type) {
    // an output is its own input's memory or nobody's: q's is read and written apart from k's
    if (a.tokens && a.q.heads && a.k.heads &&
        (a.oq.p == a.ok.p || a.oq.p == a.k.p || a.ok.p == a.q.p))
        return ARK_E_INVALID_ARG;
    if (!a.pos && a.seq == 0) return ARK_E_INVALID_ARG;
    if (a.pos && pos_type != ARK_TYPE_I32 && pos_type != ARK_TYPE_I64) return ARK_E_INVALID_ARG;
    if (a.pos && !aligned_to(a.pos, a.pos64 ? 8 : 4)) return ARK_E_MISALIGNED;
    if (a.tokens >= (1ull << 40)) return ARK_E_INVALID_ARG;
    if (a.oq.heads != a.q.heads || a.ok.heads != a.k.heads) return ARK_E_INVALID_ARG;
    int rc = ARK_OK;
    heads_ok(a.q, a.tokens, dim, e, false, &rc) && heads_ok(a.k, a.tokens, dim, e, false, &rc) &&
        heads_ok(a.oq, a.tokens, dim, e, true, &rc) && heads_ok(a.ok, a.tokens, dim, e, true, &rc);
    return rc;
}

// Groups that share a token's heads.  More of them level the SMs' loads, and each
// forms the token's angles again, which costs as much as one to two heads: three
// tasks for each group that fits, as long as a task keeps 8 heads; with fewer
// tokens than that, as many as fill the device, down to one head.
uint32_t splits_of(uint64_t tokens, uint64_t heads, uint32_t group) {
    const uint64_t fit = (uint64_t)sm_count() * kBlocksPerSm * (kThreads / group);
    uint64_t n = (3 * fit + tokens - 1) / tokens;
    if (n > heads / 8) n = heads / 8;
    const uint64_t fill = fit / tokens;   // without a second round
    if (n < fill) n = fill < heads ? fill : heads;
    return (uint32_t)(n ? n : 1);
}

// blocks that the tokens' tasks fill, at most `most`
uint32_t blocks_of(uint64_t tokens, uint32_t splits, uint32_t group, uint64_t most) {
    const uint64_t in_warp = 32 / group, warps = (tokens + in_warp - 1) / in_warp * splits;
    const uint64_t need = (warps + kThreads / 32 - 1) / (kThreads / 32);
    return (uint32_t)(need < most ? need : most);
}

// the static form of a head, where there is one (16-bit types)
template <class T>
int full_of(const Deal& d, int vec) {
    if (sizeof(T) != 2 || vec != 8 || d.rot != d.dim) return 0;
    return d.dim == 128 ? 8 : d.dim == 64 ? 4 : 0;
}

template <class T, int VEC, int NU, int G, bool NORM, int HOLD>
int forward_t(Args& a, cudaStream_t s) {
    a.splits = splits_of(a.tokens, a.q.heads + a.k.heads, a.d.group);
    const uint32_t grid = blocks_of(a.tokens, a.splits, a.d.group, (uint64_t)sm_count() * 16);
    forward_kernel<T, VEC, NU, G, NORM, HOLD><<<grid, kThreads, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, bool NORM, int HOLD>
int forward_v(Args& a, int vec, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        const int full = full_of<T>(a.d, vec);
        if (full == 8) return forward_t<T, 8, 1, 8, NORM, HOLD>(a, s);
        if (full == 4) return forward_t<T, 8, 1, 4, NORM, HOLD>(a, s);
    }
    if (vec == 8) return forward_t<T, 8, 1, 0, NORM, HOLD>(a, s);
    if constexpr (HOLD != 0)
        return ARK_E_UNSUPPORTED;   // not reached: the checkpoint is then a launch of its own
    else
        return vec == 4   ? forward_t<T, 4, 1, 0, NORM, 0>(a, s)
               : vec == 2 ? forward_t<T, 2, 2, 0, NORM, 0>(a, s)
                          : forward_t<T, 1, 4, 0, NORM, 0>(a, s);
}

template <class T, int VEC, int NU, int G>
int backward_t(Args& a, uint32_t blocks, cudaStream_t s) {
    const size_t smem = (size_t)(kThreads / a.d.group) * a.d.dim * sizeof(float);
    if (a.kind < 0)
        backward_kernel<T, VEC, NU, G, 0><<<blocks, kThreads, smem, s>>>(a);
    else if (a.kind == kE4M3)
        backward_kernel<T, VEC, NU, G, 1 + kE4M3><<<blocks, kThreads, smem, s>>>(a);
    else
        backward_kernel<T, VEC, NU, G, 1 + kInt8><<<blocks, kThreads, smem, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

// Blocks of the backward: those that fit, shared between queries and keys
// by their heads, and none without a task.
uint32_t back_blocks(Args& a) {
    const uint64_t hq = a.q.heads, hk = a.k.heads, most = (uint64_t)sm_count() * kBackPerSm;
    const uint64_t tokens = a.tokens ? a.tokens : 1;   // no tokens: a block without work leaves zero sums
    a.q_splits = splits_of(tokens, hq, a.d.group);
    a.k_splits = splits_of(tokens, hk, a.d.group);
    uint64_t bq = hq ? most * hq / (hq + hk) : 0, bk = hk ? most - bq : 0;
    if (hq && !bq) bq = 1;
    if (hk && !bk) bk = 1;
    a.q_blocks = hq ? blocks_of(tokens, a.q_splits, a.d.group, bq) : 0;
    return a.q_blocks + (hk ? blocks_of(tokens, a.k_splits, a.d.group, bk) : 0);
}

void fill_positions(Args& a, const void* positions, int32_t type, uint64_t seq) {
    a.pos = positions;
    a.pos64 = type == ARK_TYPE_I64;
    a.seq = seq;
}

int held_ok(const ark_act8* c, const Heads& h, uint64_t tokens, uint64_t dim) {
    const int rc = act8_check(c);
    if (rc) return rc;
    return c->rows == tokens && c->cols == h.heads * dim ? ARK_OK : ARK_E_INVALID_ARG;
}

}  // namespace
}  // namespace ark

using namespace ark;

extern "C" {

int ark_cuda_rope_plan(ark_rope_plan* out, uint32_t rotary_dim, uint32_t interleaved, double base,
                       uint32_t scaling, double factor, double original, double fast, double slow) {
    if (!out || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > kMaxDim || interleaved > 1 ||
        !(base > 1.0) || !isfinite(base) || scaling > ARK_ROPE_WAVE)
        return ARK_E_INVALID_ARG;
    const double pi2 = 6.283185307179586476925;
    if (scaling != ARK_ROPE_NONE && (!(factor >= 1.0) || !isfinite(factor))) return ARK_E_INVALID_ARG;
    if (scaling == ARK_ROPE_BASE) {
        if (rotary_dim == 2) return ARK_E_INVALID_ARG;
        base *= pow(factor, (double)rotary_dim / (rotary_dim - 2));
    }
    double lo = 0.0, hi = 0.0;
    if (scaling == ARK_ROPE_PARTS || scaling == ARK_ROPE_WAVE) {
        if (!(original > 0.0) || !isfinite(original) || !(slow > 0.0) || !(fast > slow) || !isfinite(fast))
            return ARK_E_INVALID_ARG;
        if (scaling == ARK_ROPE_PARTS) {
            // pairs that make `fast` and `slow` turns over the original length
            lo = floor(rotary_dim * log(original / (fast * pi2)) / (2.0 * log(base)));
            hi = ceil(rotary_dim * log(original / (slow * pi2)) / (2.0 * log(base)));
            if (lo < 0.0) lo = 0.0;
            if (hi > rotary_dim - 1.0) hi = rotary_dim - 1.0;
        }
    }
    memset(out, 0, sizeof(*out));
    out->rotary_dim = rotary_dim;
    out->interleaved = interleaved;
    out->gain = scaling == ARK_ROPE_PARTS ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        double w = pow(base, -2.0 * i / rotary_dim);   // radians per position
        if (scaling == ARK_ROPE_LINEAR) {
            w /= factor;
        } else if (scaling == ARK_ROPE_PARTS) {
            const double span = hi - lo > 0.001 ? hi - lo : 0.001;
            double ramp = (i - lo) / span;
            ramp = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
            w = w / factor * ramp + w * (1.0 - ramp);
        } else if (scaling == ARK_ROPE_WAVE) {
            double keep = (original * w / pi2 - slow) / (fast - slow);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            w = w * keep + w / factor * (1.0 - keep);
        }
        out->turns[i] = (uint64_t)ldexp(w / pi2, 64);   // w <= 1: below a sixth of a turn
    }
    return ARK_OK;
}

int ark_cuda_rope(const ark_rope_plan* plan, const ark_heads* q, const ark_heads* k,
                  const ark_heads* out_q, const ark_heads* out_k, int32_t type, uint64_t tokens,
                  uint64_t dim, const void* positions, int32_t pos_type, uint64_t seq_len,
                  int32_t inverse, void* cuda_stream) {
    int rc = plan_ok(plan, dim);
    if (rc) return rc;
    const uint64_t e = type_size(type);
    if (!e || !q || !out_q || (!k != !out_k)) return ARK_E_INVALID_ARG;
    Args a;
    memset(&a, 0, sizeof(a));
    a.plan = *plan;
    fill_positions(a, positions, pos_type, seq_len);
    a.inverse = inverse != 0;
    a.tokens = tokens;
    a.q = heads_of(q), a.k = heads_of(k), a.oq = heads_of(out_q), a.ok = heads_of(out_k);
    a.kind = -1;
    rc = common_ok(a, e, dim, pos_type);
    if (rc) return rc;
    if (tokens == 0 || a.q.heads + a.k.heads == 0) return ARK_OK;
    const Heads all[4] = {a.q, a.k, a.oq, a.ok};
    const int vec = chunk_of(plan, dim, e, all, 4);
    a.d = deal_of(plan, dim, vec);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return by_type(type, [&](auto t) { return forward_v<decltype(t), false, 0>(a, vec, s); });
}

int ark_cuda_qk_norm_rope(const ark_rope_plan* plan, const ark_heads* q, const ark_heads* k,
                          const ark_heads* out_q, const ark_heads* out_k, int32_t type,
                          uint64_t tokens, uint64_t dim, const void* gain_q, const void* gain_k,
                          int32_t gain_type, float eps, const void* positions, int32_t pos_type,
                          uint64_t seq_len, const ark_act8* q8, const ark_act8* k8,
                          void* cuda_stream) {
    int rc = plan_ok(plan, dim);
    if (rc) return rc;
    const uint64_t e = type_size(type);
    if (!e || !type_size(gain_type) || !q || !out_q || (!k != !out_k) || !(eps >= 0.0f))
        return ARK_E_INVALID_ARG;
    Args a;
    memset(&a, 0, sizeof(a));
    a.plan = *plan;
    fill_positions(a, positions, pos_type, seq_len);
    a.tokens = tokens;
    a.q = heads_of(q), a.k = heads_of(k), a.oq = heads_of(out_q), a.ok = heads_of(out_k);
    a.gq = gain_q, a.gk = gain_k, a.gain_type = gain_type, a.eps = eps;
    a.kind = -1;
    rc = common_ok(a, e, dim, pos_type);
    if (rc) return rc;
    if ((a.q.heads && !gain_q) || (a.k.heads && !gain_k)) return ARK_E_INVALID_ARG;
    if (!aligned_to(gain_q, type_size(gain_type)) || !aligned_to(gain_k, type_size(gain_type)))
        return ARK_E_MISALIGNED;
    if (q8) {
        if (k && !k8) return ARK_E_INVALID_ARG;
        rc = held_ok(q8, a.q, tokens, dim);
        if (!rc && k) rc = held_ok(k8, a.k, tokens, dim);
        if (rc) return rc;
        if (k && k8->kind != q8->kind) return ARK_E_INVALID_ARG;
    } else if (k8) {
        return ARK_E_INVALID_ARG;
    }
    if (tokens == 0 || a.q.heads + a.k.heads == 0) return ARK_OK;
    const Heads all[4] = {a.q, a.k, a.oq, a.ok};
    const int vec = chunk_of(plan, dim, e, all, 4);
    a.d = deal_of(plan, dim, vec);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (q8) {
        a.q8 = q8->data, a.sq = q8->scale, a.pq = act8_pitch(q8->cols);
        if (k) a.k8 = k8->data, a.sk = k8->scale, a.pk = act8_pitch(k8->cols);
        // a scale block lies in one head and in the chunks of lanes side by side
        const uint32_t rot = plan->rotary_dim;
        if (vec == 8 && dim % 32 == 0 && rot % (plan->interleaved ? 32 : 64) == 0)
            return by_type(type, [&](auto t) {
                using T = decltype(t);
                return q8->kind == kE4M3 ? forward_v<T, true, 1 + kE4M3>(a, vec, s)
                                         : forward_v<T, true, 1 + kInt8>(a, vec, s);
            });
        // else a launch of its own before x may be overwritten; heads side by side
        if ((a.q.heads > 1 && a.q.hs != dim) || (a.k.heads > 1 && a.k.hs != dim))
            return ARK_E_UNSUPPORTED;
        rc = ark_cuda_act8_pack(a.q.p, type, a.q.ts, q8, cuda_stream);
        if (!rc && k) rc = ark_cuda_act8_pack(a.k.p, type, a.k.ts, k8, cuda_stream);
        if (rc) return rc;
    }
    return by_type(type, [&](auto t) { return forward_v<decltype(t), true, 0>(a, vec, s); });
}

uint64_t ark_cuda_qk_norm_rope_workspace(uint64_t dim) {
    return ((uint64_t)sm_count() * kBackPerSm + 2) * dim * sizeof(float);
}

int ark_cuda_qk_norm_rope_backward(const ark_rope_plan* plan, const ark_heads* dq,
                                   const ark_heads* dk, const ark_heads* out_dq,
                                   const ark_heads* out_dk, int32_t type, uint64_t tokens,
                                   uint64_t dim, const ark_act8* q8, const ark_act8* k8,
                                   const ark_heads* q, const ark_heads* k, const void* gain_q,
                                   const void* gain_k, int32_t gain_type, float eps,
                                   const void* positions, int32_t pos_type, uint64_t seq_len,
                                   void* dgain_q, void* dgain_k, int32_t dgain_type,
                                   int32_t accumulate, void* workspace, uint64_t workspace_bytes,
                                   void* cuda_stream) {
    int rc = plan_ok(plan, dim);
    if (rc) return rc;
    const uint64_t e = type_size(type);
    if (!e || !type_size(gain_type) || !type_size(dgain_type) || !dq || !out_dq ||
        (!dk != !out_dk) || !(eps >= 0.0f) || (!q8 == !q) || (dk && (!k8 == !k)) ||
        (dk && !q8 != !k8))
        return ARK_E_INVALID_ARG;
    Args a;
    memset(&a, 0, sizeof(a));
    a.plan = *plan;
    fill_positions(a, positions, pos_type, seq_len);
    a.inverse = 1;
    a.tokens = tokens;
    a.q = heads_of(dq), a.k = heads_of(dk), a.oq = heads_of(out_dq), a.ok = heads_of(out_dk);
    a.xq = heads_of(q), a.xk = heads_of(dk ? k : nullptr);
    a.gq = gain_q, a.gk = gain_k, a.gain_type = gain_type, a.eps = eps;
    a.kind = -1;
    rc = common_ok(a, e, dim, pos_type);
    if (rc) return rc;
    if (q8) {
        rc = held_ok(q8, a.q, tokens, dim);
        if (!rc && dk) rc = held_ok(k8, a.k, tokens, dim);
        if (rc) return rc;
        if (dk && k8->kind != q8->kind) return ARK_E_INVALID_ARG;
        a.kind = q8->kind;
        a.q8 = q8->data, a.sq = q8->scale, a.pq = act8_pitch(q8->cols);
        if (dk) a.k8 = k8->data, a.sk = k8->scale, a.pk = act8_pitch(k8->cols);
    } else {
        if (a.xq.heads != a.q.heads || a.xk.heads != a.k.heads) return ARK_E_INVALID_ARG;
        if (!heads_ok(a.xq, tokens, dim, e, false, &rc) || !heads_ok(a.xk, tokens, dim, e, false, &rc))
            return rc;
    }
    if ((a.q.heads && (!gain_q || !dgain_q)) || (a.k.heads && (!gain_k || !dgain_k)))
        return ARK_E_INVALID_ARG;
    if (dk && dgain_q && dgain_q == dgain_k) return ARK_E_INVALID_ARG;
    if (!aligned_to(gain_q, type_size(gain_type)) || !aligned_to(gain_k, type_size(gain_type)) ||
        !aligned_to(dgain_q, type_size(dgain_type)) || !aligned_to(dgain_k, type_size(dgain_type)))
        return ARK_E_MISALIGNED;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (!dk) dgain_k = nullptr;
    auto sum_gains = [&](uint32_t blocks) {
        gains_kernel<<<(2 * (unsigned)dim * 32 + kThreads - 1) / kThreads, kThreads, 0, s>>>(
            a.partial, a.q_blocks, blocks, (uint32_t)dim, dgain_q, dgain_k, dgain_type, accumulate != 0);
        return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
    };
    if (a.q.heads + a.k.heads == 0) return accumulate || (!dgain_q && !dgain_k) ? ARK_OK : sum_gains(0);
    if (!workspace || workspace_bytes < ark_cuda_qk_norm_rope_workspace(dim)) return ARK_E_INVALID_ARG;
    if (!aligned_to(workspace, 4)) return ARK_E_MISALIGNED;
    a.partial = static_cast<float*>(workspace);
    const Heads all[6] = {a.q, a.k, a.oq, a.ok, a.xq, a.xk};
    const int vec = chunk_of(plan, dim, e, all, 6);
    a.d = deal_of(plan, dim, vec);
    const uint32_t blocks = back_blocks(a);
    rc = by_type(type, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2) {
            const int full = full_of<T>(a.d, vec);
            if (full == 8) return backward_t<T, 8, 1, 8>(a, blocks, s);
            if (full == 4) return backward_t<T, 8, 1, 4>(a, blocks, s);
        }
        return vec == 8   ? backward_t<T, 8, 1, 0>(a, blocks, s)
               : vec == 4 ? backward_t<T, 4, 1, 0>(a, blocks, s)
               : vec == 2 ? backward_t<T, 2, 2, 0>(a, blocks, s)
                          : backward_t<T, 1, 4, 0>(a, blocks, s);
    });
    return rc ? rc : sum_gains(blocks);
}

}  // extern "C"
