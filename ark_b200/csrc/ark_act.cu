// ark_act.cu -- 8-bit activation checkpoints (pack, unpack) and SwiGLU with
// its backward from them.  All four kernels stream: every element is read
// and written once and a column block's scale is formed in registers.
//
// One thread holds 16 consecutive columns, so 2 neighbouring lanes hold the 32
// columns of a scale block and one shuffle gives its largest magnitude.  A row
// has pitch/16 such chunks, a multiple of 8, so a scale block never straddles
// two warps; the padded columns are chunks like the others that read as zero.
// HBM and the instructions per element are near each other here (FP16, 11008
// columns: packing 72 % of the HBM's cycles and 50 % of the issue slots, SwiGLU with
// checkpoints 61 and 62, its backward 62 and 69, with the product remade 45 and
// 75), so the 16-bit types keep to pairs: the largest magnitude by integer maxima of
// two, and FP16 is scaled and rounded to 8 bits as FP16 pairs where the block's
// scale is an FP16 number.
#include "ark_act8.cuh"

namespace ark {

int act8_check(const ark_act8* c) {
    if (!c) return ARK_E_INVALID_ARG;
    if (c->kind != ARK_ACT8_E4M3 && c->kind != ARK_ACT8_INT8) return ARK_E_INVALID_ARG;
    if (c->cols >= (1ull << 31) || c->rows >= (1ull << 40)) return ARK_E_INVALID_ARG;
    if (c->rows == 0 || c->cols == 0) return ARK_OK;
    if (!c->data || !c->scale) return ARK_E_INVALID_ARG;
    if (!aligned_to(c->data, 16) || !aligned_to(c->scale, 4)) return ARK_E_MISALIGNED;
    return ARK_OK;
}

namespace {

constexpr int kThreads = 256;

// Place (row, chunk) of a thread in a grid-stride walk over rows * per_row
// chunks: one division at the start, none in the loop.
struct Walk {
    uint64_t row, drow;
    uint32_t chunk, dchunk, per_row;
    __device__ Walk(uint64_t i, uint64_t stride, uint32_t per) : per_row(per) {
        row = i / per;
        chunk = (uint32_t)(i - row * per);
        drow = stride / per;
        dchunk = (uint32_t)(stride - drow * per);
    }
    __device__ __forceinline__ void next() {
        row += drow;
        chunk += dchunk;
        if (chunk >= per_row) {
            chunk -= per_row;
            ++row;
        }
    }
};

// columns of a row from col on, as far as a thread asks (32)
__device__ __forceinline__ int left(uint32_t cols, uint32_t col) {
    return col < cols ? (int)min(cols - col, 32u) : 0;
}

// ------------------------------------------------------------ words of a thread
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {   // 32-byte aligned
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                   "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ void load16(const void* p, uint32_t* w) {
    const uint4 q = *static_cast<const uint4*>(p);
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
}
__device__ __forceinline__ void store16(void* p, const uint32_t* w) {
    *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// W + 4 words, of which the W from byte `by` (0 to 16) on come to the front
template <int W>
__device__ __forceinline__ void shift(uint32_t* v, uint32_t by) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = by & 16 ? v[i + 4] : v[i];
#pragma unroll
    for (int i = 0; i < W + 2; ++i) v[i] = by & 8 ? v[i + 2] : v[i];
#pragma unroll
    for (int i = 0; i < W + 1; ++i) v[i] = by & 4 ? v[i + 1] : v[i];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = by & 2 ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
}

// How a tensor's rows lie: kStraight32 / kStraight16: every row starts on a 32- /
// 16-byte boundary; kAny: on any element.  The last is served by whole 16-byte
// vectors too, shifted in registers: a thread reads the vectors around its
// columns where those lie inside the row, and writes whole vectors with the end
// of its neighbour's columns, which it gets by a shuffle (2-byte accesses 32
// bytes apart took 570 us where this takes 62: unpack, 8192 x 11003 to FP16).
enum Lie { kAny, kStraight16, kStraight32 };

template <int W>
__device__ __forceinline__ bool load_words(const void* p, uint32_t col, int n, int lie, uint32_t* w) {
    if (lie == kStraight32 && n >= 16) {
#pragma unroll
        for (int i = 0; i < W; i += 8) load32(static_cast<const uint32_t*>(p) + i, w + i);
        return true;
    }
    if (lie == kStraight16 && n >= 16) {
#pragma unroll
        for (int i = 0; i < W; i += 4) load16(static_cast<const uint32_t*>(p) + i, w + i);
        return true;
    }
    // 8 columns to each side are the row's
    if (lie == kAny && col > 0 && n >= 24) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
        const char* from = static_cast<const char*>(p) - off;
        uint32_t v[W + 4];
#pragma unroll
        for (int i = 0; i < W; i += 4) load16(from + 4 * i, v + i);
        v[W] = v[W + 1] = v[W + 2] = v[W + 3] = 0;
        if (off) load16(from + 4 * W, v + W);
        shift<W>(v, off);
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = v[i];
        return true;
    }
    return false;
}
// All lanes of a warp take part.  E: bytes of an element.
template <int W, int E>
__device__ __forceinline__ void store_words(void* p, uint32_t col, int n, int lie, const uint32_t* w) {
    char* q = static_cast<char*>(p);
    auto some = [&](int lo, int hi) {   // elements lo to hi - 1, one by one
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i >= lo && i < hi) {
                if (E == 4)
                    reinterpret_cast<uint32_t*>(q)[i] = w[i];
                else
                    reinterpret_cast<uint16_t*>(q)[i] = i & 1 ? hi16(w[i >> 1]) : lo16(w[i >> 1]);
            }
    };
    if (lie != kAny) {
        if (n < 16) {
            some(0, n);
        } else if (lie == kStraight32) {
#pragma unroll
            for (int i = 0; i < W; i += 8) store32(q + 4 * i, w + i);
        } else {
#pragma unroll
            for (int i = 0; i < W; i += 4) store16(q + 4 * i, w + i);
        }
        return;
    }
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(q) & 15u);
    const int lane = threadIdx.x & 31;
    const bool whole = n >= 16;
    // the lane before holds the columns before mine, whole; the same behind me
    const uint32_t wholes = __ballot_sync(0xFFFFFFFFu, whole);
    const uint32_t starts = __ballot_sync(0xFFFFFFFFu, col == 0);
    const bool before = lane > 0 && (wholes >> (lane - 1) & 1) && col > 0;
    const bool behind = lane < 31 && (wholes >> (lane + 1) & 1) && !(starts >> (lane + 1) & 1);
    uint32_t v[W + 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __shfl_up_sync(0xFFFFFFFFu, w[W - 4 + i], 1);
#pragma unroll
    for (int i = 0; i < W; ++i) v[4 + i] = w[i];
    if (!whole) {
        some(0, n);
        return;
    }
    shift<W>(v, 16 - off);
    const bool head = off == 0 || before;   // all of the first vector is known
#pragma unroll
    for (int i = 0; i < W; i += 4)
        if (i > 0 || head) store16(q - off + 4 * i, v + i);
    if (!head) some(0, (int)(16 - off) / E);
    if (off && !behind) some(16 - (int)off / E, 16);
}

// ------------------------------------------------------------ 16 columns of a thread
template <class T>
struct Chunk {   // a 16-bit type: pairs
    uint32_t w[8];

    __device__ __forceinline__ void load(const T* p, uint32_t col, int n, int lie) {
        if (load_words<8>(p + col, col, n, lie, w)) return;
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + col;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = pack16(2 * i < n ? q[2 * i] : (uint16_t)0, 2 * i + 1 < n ? q[2 * i + 1] : (uint16_t)0);
    }
    __device__ __forceinline__ void store(T* p, uint32_t col, int n, int lie) const {
        store_words<8, 2>(p + col, col, n, lie, w);
    }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) widen2(w[i], v[2 * i], v[2 * i + 1], T());
    }
    __device__ __forceinline__ void set(const float* v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = narrow2(v[2 * i], v[2 * i + 1], T());
    }
    // FP32 bits of the largest magnitude of the block that two lanes hold
    __device__ __forceinline__ uint32_t block_max() const {
        uint32_t m = pairs_max<8>(w);
        m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        return pairs_bits(m, T());
    }
    template <int KIND>
    __device__ __forceinline__ uint4 quant(uint32_t byte) const {
        uint32_t o[4];
        quant_words<T, KIND, 8>(w, byte, o);
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};
template <>
struct Chunk<float> {
    float f[16];

    __device__ __forceinline__ void load(const float* p, uint32_t col, int n, int lie) {
        uint32_t w[16];
        if (load_words<16>(p + col, col, n, lie, w)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(w[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = i < n ? p[col + i] : 0.0f;
    }
    __device__ __forceinline__ void store(float* p, uint32_t col, int n, int lie) const {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(f[i]);
        store_words<16, 4>(p + col, col, n, lie, w);
    }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = f[i];
    }
    __device__ __forceinline__ void set(const float* v) {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = v[i];
    }
    __device__ __forceinline__ uint32_t block_max() const {
        const uint32_t m = abs_max<16>(f);
        return max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    }
    template <int KIND>
    __device__ __forceinline__ uint4 quant(uint32_t byte) const {
        if (byte == kActBad) return make_uint4(0u, 0u, 0u, 0u);
        const float inv = inv_scale(byte);
        return make_uint4(quant4<KIND>(f, inv), quant4<KIND>(f + 4, inv), quant4<KIND>(f + 8, inv),
                          quant4<KIND>(f + 12, inv));
    }
};

// one thread's 16 columns of a checkpoint; all lanes of a warp take part
template <int KIND, class T>
__device__ __forceinline__ void hold(uint8_t* data, uint8_t* scale, uint64_t chunk, bool on,
                                     const Chunk<T>& c) {
    const uint32_t byte = scale_byte<KIND>(c.block_max());
    if (!on) return;
    *reinterpret_cast<uint4*>(data + chunk * 16) = c.template quant<KIND>(byte);
    if ((threadIdx.x & 1) == 0) scale[chunk >> 1] = (uint8_t)byte;
}

// 16 stored columns as FP32
template <int KIND>
__device__ __forceinline__ void held(const uint8_t* data, const uint8_t* scale, uint64_t chunk,
                                     float* v) {
    const uint4 q = *reinterpret_cast<const uint4*>(data + chunk * 16);
    const uint32_t byte = scale[chunk >> 1];
    dequant8<KIND>(make_uint2(q.x, q.y), byte, v);
    dequant8<KIND>(make_uint2(q.z, q.w), byte, v + 8);
}

// ------------------------------------------------------------ pack, unpack
template <class T, int KIND>
__global__ void __launch_bounds__(kThreads) pack_kernel(const T* __restrict__ x, uint64_t ldx,
                                                        uint64_t rows, uint32_t cols,
                                                        uint32_t per_row, int lie,
                                                        uint8_t* __restrict__ data,
                                                        uint8_t* __restrict__ scale) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;   // a multiple of 8: lanes of a block leave together
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        Chunk<T> c;
        c.load(x + w.row * ldx, w.chunk * 16, i < total ? left(cols, w.chunk * 16) : 0, lie);
        hold<KIND>(data, scale, i, i < total, c);
    }
}

// OPERAND: as operand16 says
template <class T, int KIND, bool OPERAND = false>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const uint8_t* __restrict__ data,
                                                          const uint8_t* __restrict__ scale,
                                                          uint64_t rows, uint32_t cols,
                                                          uint32_t per_row, int lie,
                                                          T* __restrict__ y, uint64_t ldy) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        const uint32_t col = w.chunk * 16;
        const int n = i < total ? left(cols, col) : 0;
        const uint64_t at = i < total ? i : 0;
        Chunk<T> c;
        if constexpr (std::is_same<T, float>::value) {
            held<KIND>(data, scale, at, c.f);
#pragma unroll
            for (int j = 0; j < 16; ++j) c.f[j] = saturate<float>(c.f[j]);
        } else {
            uint4 lo, hi;
            operand16<T, KIND, OPERAND>(*reinterpret_cast<const uint4*>(data + at * 16), scale[at >> 1],
                                        lo, hi);
            c.w[0] = lo.x, c.w[1] = lo.y, c.w[2] = lo.z, c.w[3] = lo.w;
            c.w[4] = hi.x, c.w[5] = hi.y, c.w[6] = hi.z, c.w[7] = hi.w;
        }
        c.store(y + w.row * ldy, col, n, lie);
    }
}

// 16-bit rows from any boundary to 16-byte ones
__global__ void __launch_bounds__(kThreads) realign_kernel(const __half* __restrict__ src, uint64_t ld,
                                                           uint64_t rows, uint32_t cols,
                                                           uint32_t per_row, __half* __restrict__ dst,
                                                           uint64_t ldd) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads, total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; i < total; i += stride, w.next()) {
        const uint32_t col = w.chunk * 16;
        Chunk<__half> c;
        c.load(src + w.row * ld, col, left(cols, col), kAny);
        c.store(dst + w.row * ldd, col, left(cols, col), kStraight16);
    }
}

// ------------------------------------------------------------ SwiGLU
// silu(a) = a * s with s = 1 / (1 + exp(-a)); its slope is s * (1 + a * (1 - s)).
// From e = exp(-|a|) <= 1, which can underflow but not overflow, both s and
// 1 - s come without cancellation and keep their small end.
// T: what the result is rounded to.  For a 16-bit type the fast exponential, off by
// 2 + 1.2 |a| ulps of FP32, is far below its half step; FP32 results take the full one
// (1 ulp).  The reciprocal is off by 1.
template <class T>
__device__ __forceinline__ void sigmoid(float a, float& s, float& rest) {
    const float e = std::is_same<T, float>::value ? expf(-fabsf(a)) : __expf(-fabsf(a));
    float r;   // of 1 to 2
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, e)));
    const float t = __fmul_rn(e, r);
    s = a < 0.0f ? t : r;
    rest = a < 0.0f ? r : t;
}

template <class T, int KIND, bool HOLD>
__global__ void __launch_bounds__(kThreads) swiglu_kernel(
    const T* a, uint64_t lda, const T* b, uint64_t ldb, uint64_t rows, uint32_t cols,
    uint32_t per_row, int lie, T* y, uint64_t ldy, uint8_t* __restrict__ a8,
    uint8_t* __restrict__ sa, uint8_t* __restrict__ b8, uint8_t* __restrict__ sb) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        const uint32_t col = w.chunk * 16;
        const int n = i < total ? left(cols, col) : 0;
        Chunk<T> ca, cb, cy;
        ca.load(a + w.row * lda, col, n, lie);
        cb.load(b + w.row * ldb, col, n, lie);
        float u[16], v[16];
        ca.get(u);
        cb.get(v);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float s, rest;
            sigmoid<T>(u[j], s, rest);
            u[j] = __fmul_rn(__fmul_rn(u[j], s), v[j]);
        }
        cy.set(u);
        cy.store(y + w.row * ldy, col, n, lie);
        if (HOLD) {
            hold<KIND>(a8, sa, i, i < total, ca);
            hold<KIND>(b8, sb, i, i < total, cb);
        }
    }
}

// One stored element in 64 bits.
template <int KIND>
__device__ __forceinline__ double held_one(const uint8_t* data, const uint8_t* scale, uint64_t at) {
    float v[4];
    bytes4<KIND>(data[at], v);
    return (double)__fmul_rn(v[0], scale_of(scale[at >> 5]));
}
// Whether y rounds to two values of T when it is off by a factor of up to `most`.
template <class T>
__device__ __forceinline__ bool splits(float y, float most) {
    const uint32_t w = narrow2(__fmul_rn(y, most), __fmul_rn(y, __fsub_rn(2.0f, most)), T());
    return __byte_perm(w, w, 0x1032) != w;
}

// With y8, the product is remade, rounded to T as the forward's was, and
// checkpointed for the weight gradient of the projection that read it.  The
// product of two 8-bit values often lies next to a border of T, and once rounded
// next to one of the 8-bit grid, where the last bit of FP32 would decide by a whole
// step: values within FP32's error of a border of T, about one in 500, are made
// again in 64 bits and rounded to FP32.  Rounding both ends of the error finds the
// borders of every size, those of FP16's subnormals too.  An FP32 product is packed as
// FP32 made it: next to a border of the 8-bit grid it may go either way.
// Blocks an SM: what 80 and 64 registers allow, without spills.
template <class T, int KIND, bool REMAKE>
__global__ void __launch_bounds__(kThreads, REMAKE ? 3 : 4) swiglu_back_kernel(
    const T* dy, uint64_t lddy, const uint8_t* __restrict__ a8, const uint8_t* __restrict__ sa,
    const uint8_t* __restrict__ b8, const uint8_t* __restrict__ sb, uint64_t rows, uint32_t cols,
    uint32_t per_row, int lie, T* da, uint64_t ldda, T* db, uint64_t lddb,
    uint8_t* __restrict__ y8, uint8_t* __restrict__ sy) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        const uint32_t col = w.chunk * 16;
        const int n = i < total ? left(cols, col) : 0;
        const uint64_t at = i < total ? i : 0;
        Chunk<T> g, cy;
        g.load(dy + w.row * lddy, col, n, lie);
        float u[16], v[16], d[16], o[16];
        uint32_t near = 0;
        held<KIND>(a8, sa, at, u);
        held<KIND>(b8, sb, at, v);
        g.get(d);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float s, rest;
            sigmoid<T>(u[j], s, rest);
            const float t = __fmul_rn(u[j], s);
            const float slope = __fmul_rn(s, __fmaf_rn(u[j], rest, 1.0f));
            o[j] = __fmul_rn(t, v[j]);
            if constexpr (REMAKE && !std::is_same<T, float>::value) {
                // exp(-|a|) is off by 2 + 1.2 |a| ulps of 2^-23, of which `rest` reaches s;
                // the sum, the reciprocal and three products add 4, the test itself 1
                constexpr float kUlp = 1.0f / 8388608.0f;
                const float most = __fmaf_rn(__fmaf_rn(1.2f * kUlp, fabsf(u[j]), 2 * kUlp), rest,
                                             1.0f + 5 * kUlp);
                near |= splits<T>(o[j], most) ? 1u << j : 0u;
            }
            u[j] = __fmul_rn(__fmul_rn(d[j], v[j]), slope);
            v[j] = __fmul_rn(d[j], t);
        }
        g.set(u);
        g.store(da + w.row * ldda, col, n, lie);
        g.set(v);
        g.store(db + w.row * lddb, col, n, lie);
        if (REMAKE) {
            if constexpr (!std::is_same<T, float>::value) {
                for (; near; near &= near - 1) {
                    const int which = __ffs(near) - 1;
                    const double p = held_one<KIND>(a8, sa, at * 16 + which);
                    const double q = held_one<KIND>(b8, sb, at * 16 + which);
                    const float y = (float)(p / (1.0 + exp(-p)) * q);
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = j == which ? y : o[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = j < n ? o[j] : 0.0f;
            cy.set(o);
            hold<KIND>(y8, sy, i, i < total, cy);
        }
    }
}

template <class T>
int lie_of(const T* p, uint64_t ld) {
    return aligned_to(p, 32) && ld * sizeof(T) % 32 == 0 ? kStraight32
           : aligned16(p) && ld * sizeof(T) % 16 == 0    ? kStraight16
                                                         : kAny;
}
int least(int a, int b) { return a < b ? a : b; }

// rows of cols elements, ld apart
bool shape_ok(uint64_t rows, uint64_t cols, uint64_t ld) {
    return cols < (1ull << 31) && rows < (1ull << 40) && (rows <= 1 || ld >= cols || ld == 0);
}

// At most 8 blocks of 256 threads an SM.  Packing (32 registers) has them all resident;
// unpacking holds 6, SwiGLU 3 with checkpoints (71 to 80 registers) and 4 in the
// backward (64), so that a grid of 8 runs in rounds there.
unsigned grid_of(uint64_t work) {
    const uint64_t need = (work + kThreads - 1) / kThreads, most = (uint64_t)sm_count() * 8;
    return (unsigned)(need < most ? need : most);
}

template <class T, int KIND>
int pack_t(const T* x, uint64_t ldx, const ark_act8* o, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(o->cols) / 16);
    auto k = pack_kernel<T, KIND>;
    k<<<grid_of(o->rows * per), kThreads, 0, s>>>(x, ldx, o->rows, (uint32_t)o->cols, per,
                                                     lie_of(x, ldx), o->data, o->scale);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND, bool OPERAND = false>
int unpack_t(const ark_act8* c, T* y, uint64_t ldy, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(c->cols) / 16);
    auto k = unpack_kernel<T, KIND, OPERAND>;
    k<<<grid_of(c->rows * per), kThreads, 0, s>>>(c->data, c->scale, c->rows, (uint32_t)c->cols,
                                                     per, lie_of(y, ldy), y, ldy);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND, bool HOLD>
int swiglu_t(const T* a, uint64_t lda, const T* b, uint64_t ldb, uint64_t rows, uint64_t cols, T* y,
             uint64_t ldy, const ark_act8* a8, const ark_act8* b8, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(cols) / 16);
    const int lie = least(least(lie_of(a, lda), lie_of(b, ldb)), lie_of(y, ldy));
    auto k = swiglu_kernel<T, KIND, HOLD>;
    k<<<grid_of(rows * per), kThreads, 0, s>>>(
        a, lda, b, ldb, rows, (uint32_t)cols, per, lie, y, ldy, HOLD ? a8->data : nullptr,
        HOLD ? a8->scale : nullptr, HOLD ? b8->data : nullptr, HOLD ? b8->scale : nullptr);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND, bool REMAKE>
int swiglu_back_t(const T* dy, uint64_t lddy, const ark_act8* a8, const ark_act8* b8, T* da,
                  uint64_t ldda, T* db, uint64_t lddb, const ark_act8* y8, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(a8->cols) / 16);
    const int lie = least(least(lie_of(dy, lddy), lie_of(da, ldda)), lie_of(db, lddb));
    auto k = swiglu_back_kernel<T, KIND, REMAKE>;
    k<<<grid_of(a8->rows * per), kThreads, 0, s>>>(
        dy, lddy, a8->data, a8->scale, b8->data, b8->scale, a8->rows, (uint32_t)a8->cols, per, lie,
        da, ldda, db, lddb, REMAKE ? y8->data : nullptr, REMAKE ? y8->scale : nullptr);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

bool same_shape(const ark_act8* a, const ark_act8* b) {
    return a->rows == b->rows && a->cols == b->cols && a->kind == b->kind;
}

}  // namespace

int act8_operands(const ark_act8* c, void* y, int32_t type, uint64_t ldy, cudaStream_t s) {
    if (type == ARK_TYPE_F16) {
        __half* p = static_cast<__half*>(y);
        return c->kind == kE4M3 ? unpack_t<__half, kE4M3, true>(c, p, ldy, s)
                                : unpack_t<__half, kInt8, true>(c, p, ldy, s);
    }
    // BF16 operands are what unpacking makes
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(y);
    return c->kind == kE4M3 ? unpack_t<__nv_bfloat16, kE4M3>(c, p, ldy, s)
                            : unpack_t<__nv_bfloat16, kInt8>(c, p, ldy, s);
}

int realign_rows(const void* src, uint64_t ld, uint64_t rows, uint32_t cols, void* dst, uint64_t ldd,
                 cudaStream_t s) {
    const uint32_t per = (cols + 15) / 16;
    realign_kernel<<<grid_of(rows * per), kThreads, 0, s>>>(
        static_cast<const __half*>(src), ld, rows, cols, per, static_cast<__half*>(dst), ldd);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

}  // namespace ark

using namespace ark;

extern "C" {

uint64_t ark_cuda_act8_pitch(uint64_t cols) { return act8_pitch(cols); }

int ark_cuda_act8_pack(const void* x, int32_t type, uint64_t ldx, const ark_act8* out,
                       void* cuda_stream) {
    const int rc = act8_check(out);
    if (rc) return rc;
    if (!type_size(type) || !shape_ok(out->rows, out->cols, ldx)) return ARK_E_INVALID_ARG;
    if (out->rows == 0 || out->cols == 0) return ARK_OK;
    if (!x) return ARK_E_INVALID_ARG;
    if (!aligned_to(x, type_size(type))) return ARK_E_MISALIGNED;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        const T* p = static_cast<const T*>(x);
        return out->kind == kE4M3 ? pack_t<T, kE4M3>(p, ldx, out, s)
                                  : pack_t<T, kInt8>(p, ldx, out, s);
    });
}

int ark_cuda_act8_unpack(const ark_act8* in, void* y, int32_t type, uint64_t ldy,
                         void* cuda_stream) {
    const int rc = act8_check(in);
    if (rc) return rc;
    if (!type_size(type) || !shape_ok(in->rows, in->cols, ldy) || (in->rows > 1 && ldy < in->cols))
        return ARK_E_INVALID_ARG;
    if (in->rows == 0 || in->cols == 0) return ARK_OK;
    if (!y) return ARK_E_INVALID_ARG;
    if (!aligned_to(y, type_size(type))) return ARK_E_MISALIGNED;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        T* p = static_cast<T*>(y);
        return in->kind == kE4M3 ? unpack_t<T, kE4M3>(in, p, ldy, s)
                                 : unpack_t<T, kInt8>(in, p, ldy, s);
    });
}

int ark_cuda_swiglu(const void* a, uint64_t lda, const void* b, uint64_t ldb, int32_t type,
                    uint64_t rows, uint64_t cols, void* y, uint64_t ldy, const ark_act8* a8,
                    const ark_act8* b8, void* cuda_stream) {
    if (!type_size(type) || !shape_ok(rows, cols, lda) || !shape_ok(rows, cols, ldb) ||
        !shape_ok(rows, cols, ldy) || (rows > 1 && ldy < cols) || (!a8 != !b8))
        return ARK_E_INVALID_ARG;
    if (a8) {
        int rc = act8_check(a8);
        if (!rc) rc = act8_check(b8);
        if (rc) return rc;
        if (!same_shape(a8, b8) || a8->rows != rows || a8->cols != cols) return ARK_E_INVALID_ARG;
    }
    if (rows == 0 || cols == 0) return ARK_OK;
    if (!a || !b || !y) return ARK_E_INVALID_ARG;
    const uint64_t e = type_size(type);
    if (!aligned_to(a, e) || !aligned_to(b, e) || !aligned_to(y, e)) return ARK_E_MISALIGNED;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        const T *pa = static_cast<const T*>(a), *pb = static_cast<const T*>(b);
        T* py = static_cast<T*>(y);
        if (!a8) return swiglu_t<T, kE4M3, false>(pa, lda, pb, ldb, rows, cols, py, ldy, a8, b8, s);
        return a8->kind == kE4M3
                   ? swiglu_t<T, kE4M3, true>(pa, lda, pb, ldb, rows, cols, py, ldy, a8, b8, s)
                   : swiglu_t<T, kInt8, true>(pa, lda, pb, ldb, rows, cols, py, ldy, a8, b8, s);
    });
}

int ark_cuda_swiglu_backward(const void* dy, uint64_t lddy, int32_t type, const ark_act8* a8,
                             const ark_act8* b8, void* da, uint64_t ldda, void* db, uint64_t lddb,
                             const ark_act8* y8, void* cuda_stream) {
    int rc = act8_check(a8);
    if (!rc) rc = act8_check(b8);
    if (!rc && y8) rc = act8_check(y8);
    if (rc) return rc;
    const uint64_t rows = a8->rows, cols = a8->cols;
    if (!type_size(type) || !same_shape(a8, b8) || (y8 && !same_shape(a8, y8)) ||
        !shape_ok(rows, cols, lddy) || !shape_ok(rows, cols, ldda) || !shape_ok(rows, cols, lddb) ||
        (rows > 1 && (ldda < cols || lddb < cols)))
        return ARK_E_INVALID_ARG;
    if (rows == 0 || cols == 0) return ARK_OK;
    if (!dy || !da || !db || da == db) return ARK_E_INVALID_ARG;
    const uint64_t e = type_size(type);
    if (!aligned_to(dy, e) || !aligned_to(da, e) || !aligned_to(db, e)) return ARK_E_MISALIGNED;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        const T* pg = static_cast<const T*>(dy);
        T *pa = static_cast<T*>(da), *pb = static_cast<T*>(db);
        if (a8->kind == kE4M3)
            return y8 ? swiglu_back_t<T, kE4M3, true>(pg, lddy, a8, b8, pa, ldda, pb, lddb, y8, s)
                      : swiglu_back_t<T, kE4M3, false>(pg, lddy, a8, b8, pa, ldda, pb, lddb, y8, s);
        return y8 ? swiglu_back_t<T, kInt8, true>(pg, lddy, a8, b8, pa, ldda, pb, lddb, y8, s)
                  : swiglu_back_t<T, kInt8, false>(pg, lddy, a8, b8, pa, ldda, pb, lddb, y8, s);
    });
}

}  // extern "C"
