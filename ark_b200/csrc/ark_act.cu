// ark_act.cu -- 8-bit activation checkpoints (pack, unpack) and SwiGLU with
// its backward from them.  All four kernels stream: every element is read
// and written once and a column block's scale is formed in registers, so HBM
// bounds them.
//
// One thread holds 8 consecutive columns (16 bytes of a 16-bit type), so 4
// neighbouring lanes hold the 32 columns of a scale block and two shuffles
// give its largest magnitude.  A row has pitch/8 such chunks, a multiple of
// 16, so a scale block never straddles two warps; the padded columns are
// chunks like the others that read as zero.
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

// Chunk (row, column) of a thread in a grid-stride walk over rows * per_row
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

// the largest magnitude of the block that 4 neighbouring lanes hold
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    return max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
}

// one thread's 8 columns of a checkpoint
template <int KIND>
__device__ __forceinline__ void put(uint8_t* data, uint8_t* scale, uint64_t chunk, const float* v,
                                    uint32_t byte) {
    *reinterpret_cast<uint2*>(data + chunk * 8) = quant8<KIND>(v, byte);
    if ((threadIdx.x & 3) == 0) scale[chunk >> 2] = (uint8_t)byte;
}

__device__ __forceinline__ int left(uint32_t cols, uint32_t col) {
    return col < cols ? (int)min(cols - col, 8u) : 0;
}

// ------------------------------------------------------------ pack, unpack
template <class T, int KIND>
__global__ void __launch_bounds__(kThreads) pack_kernel(const T* __restrict__ x, uint64_t ldx,
                                                        uint64_t rows, uint32_t cols,
                                                        uint32_t per_row, bool vec,
                                                        uint8_t* __restrict__ data,
                                                        uint8_t* __restrict__ scale) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;   // a multiple of 16: lanes of a block leave together
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        float v[8];
        const int n = i < total ? left(cols, w.chunk * 8) : 0;
        load8(x + w.row * ldx + w.chunk * 8, n, vec, v);
        const uint32_t byte = scale_byte<KIND>(block_max(abs_max<8>(v)));
        if (i < total) put<KIND>(data, scale, i, v, byte);
    }
}

template <class T, int KIND>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const uint8_t* __restrict__ data,
                                                          const uint8_t* __restrict__ scale,
                                                          uint64_t rows, uint32_t cols,
                                                          uint32_t per_row, bool vec,
                                                          T* __restrict__ y, uint64_t ldy) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; i < total; i += stride, w.next()) {
        const int n = left(cols, w.chunk * 8);
        if (n == 0) continue;
        float v[8];
        dequant8<KIND>(*reinterpret_cast<const uint2*>(data + i * 8), scale[i >> 2], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = saturate<T>(v[j]);
        store8(y + w.row * ldy + w.chunk * 8, n, vec, v);
    }
}

// ------------------------------------------------------------ SwiGLU
// silu(a) = a * s with s = 1 / (1 + exp(-a)); its slope is s * (1 + a * (1 - s)).
// From e = exp(-|a|) <= 1, which can underflow but not overflow, both s and
// 1 - s come without cancellation and keep their small end.
__device__ __forceinline__ void sigmoid(float a, float& s, float& rest) {
    const float e = __expf(-fabsf(a));
    const float r = __fdividef(1.0f, __fadd_rn(1.0f, e)), t = __fmul_rn(e, r);
    s = a < 0.0f ? t : r;
    rest = a < 0.0f ? r : t;
}

template <class T, int KIND, bool HOLD>
__global__ void __launch_bounds__(kThreads) swiglu_kernel(
    const T* a, uint64_t lda, const T* b, uint64_t ldb, uint64_t rows,
    uint32_t cols, uint32_t per_row, bool vec, T* y, uint64_t ldy, uint8_t* __restrict__ a8,
    uint8_t* __restrict__ sa, uint8_t* __restrict__ b8, uint8_t* __restrict__ sb) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        float u[8], v[8], o[8];
        const uint32_t col = w.chunk * 8;
        const int n = i < total ? left(cols, col) : 0;
        load8(a + w.row * lda + col, n, vec, u);
        load8(b + w.row * ldb + col, n, vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float p, rest;
            sigmoid(u[j], p, rest);
            o[j] = __fmul_rn(__fmul_rn(u[j], p), v[j]);
        }
        store8(y + w.row * ldy + col, n, vec, o);
        if (HOLD) {
            const uint32_t ba = scale_byte<KIND>(block_max(abs_max<8>(u)));
            const uint32_t bb = scale_byte<KIND>(block_max(abs_max<8>(v)));
            if (i < total) {
                put<KIND>(a8, sa, i, u, ba);
                put<KIND>(b8, sb, i, v, bb);
            }
        }
    }
}

// With y8, the product is remade, rounded to T as the forward's was, and
// checkpointed for the weight gradient of the projection that read it.
template <class T, int KIND, bool REMAKE>
__global__ void __launch_bounds__(kThreads) swiglu_back_kernel(
    const T* dy, uint64_t lddy, const uint8_t* __restrict__ a8, const uint8_t* __restrict__ sa,
    const uint8_t* __restrict__ b8, const uint8_t* __restrict__ sb, uint64_t rows, uint32_t cols,
    uint32_t per_row, bool vec, T* da, uint64_t ldda, T* db, uint64_t lddb,
    uint8_t* __restrict__ y8, uint8_t* __restrict__ sy) {
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint64_t total = rows * per_row;
    const uint64_t first = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    Walk w(first, stride, per_row);
    for (uint64_t i = first; (i & ~31ull) < total; i += stride, w.next()) {
        float u[8], v[8], g[8], o[8];
        const uint32_t col = w.chunk * 8;
        const int n = i < total ? left(cols, col) : 0;
        const uint64_t at = i < total ? i : 0;
        load8(dy + w.row * lddy + col, n, vec, g);
        dequant8<KIND>(*reinterpret_cast<const uint2*>(a8 + at * 8), sa[at >> 2], u);
        dequant8<KIND>(*reinterpret_cast<const uint2*>(b8 + at * 8), sb[at >> 2], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s, rest;
            sigmoid(u[j], s, rest);
            const float t = __fmul_rn(u[j], s);
            const float slope = __fmul_rn(s, __fmaf_rn(u[j], rest, 1.0f));
            u[j] = __fmul_rn(__fmul_rn(g[j], v[j]), slope);
            o[j] = j < n ? Elem<T>::to_f(Elem<T>::from_f(__fmul_rn(t, v[j]))) : 0.0f;
            v[j] = __fmul_rn(g[j], t);
        }
        store8(da + w.row * ldda + col, n, vec, u);
        store8(db + w.row * lddb + col, n, vec, v);
        if (REMAKE) {
            const uint32_t byte = scale_byte<KIND>(block_max(abs_max<8>(o)));
            if (i < total) put<KIND>(y8, sy, i, o, byte);
        }
    }
}

template <class T>
bool rows_vec(const T* p, uint64_t ld) {
    return aligned16(p) && ld * sizeof(T) % 16 == 0;
}

// rows of 16-byte chunks: cols elements, ld apart
bool shape_ok(uint64_t rows, uint64_t cols, uint64_t ld) {
    return cols < (1ull << 31) && rows < (1ull << 40) && (rows <= 1 || ld >= cols || ld == 0);
}

// at most the 8 blocks of 256 threads that an SM holds
unsigned grid_of(uint64_t work) {
    const uint64_t need = (work + kThreads - 1) / kThreads, most = (uint64_t)sm_count() * 8;
    return (unsigned)(need < most ? need : most);
}

template <class T, int KIND>
int pack_t(const T* x, uint64_t ldx, const ark_act8* o, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(o->cols) / 8);
    auto k = pack_kernel<T, KIND>;
    k<<<grid_of(o->rows * per), kThreads, 0, s>>>(x, ldx, o->rows, (uint32_t)o->cols, per,
                                                     rows_vec(x, ldx), o->data, o->scale);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND>
int unpack_t(const ark_act8* c, T* y, uint64_t ldy, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(c->cols) / 8);
    auto k = unpack_kernel<T, KIND>;
    k<<<grid_of(c->rows * per), kThreads, 0, s>>>(c->data, c->scale, c->rows, (uint32_t)c->cols,
                                                     per, rows_vec(y, ldy), y, ldy);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND, bool HOLD>
int swiglu_t(const T* a, uint64_t lda, const T* b, uint64_t ldb, uint64_t rows, uint64_t cols, T* y,
             uint64_t ldy, const ark_act8* a8, const ark_act8* b8, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(cols) / 8);
    const bool vec = rows_vec(a, lda) && rows_vec(b, ldb) && rows_vec(y, ldy);
    auto k = swiglu_kernel<T, KIND, HOLD>;
    k<<<grid_of(rows * per), kThreads, 0, s>>>(
        a, lda, b, ldb, rows, (uint32_t)cols, per, vec, y, ldy, HOLD ? a8->data : nullptr,
        HOLD ? a8->scale : nullptr, HOLD ? b8->data : nullptr, HOLD ? b8->scale : nullptr);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

template <class T, int KIND, bool REMAKE>
int swiglu_back_t(const T* dy, uint64_t lddy, const ark_act8* a8, const ark_act8* b8, T* da,
                  uint64_t ldda, T* db, uint64_t lddb, const ark_act8* y8, cudaStream_t s) {
    const uint32_t per = (uint32_t)(act8_pitch(a8->cols) / 8);
    const bool vec = rows_vec(dy, lddy) && rows_vec(da, ldda) && rows_vec(db, lddb);
    auto k = swiglu_back_kernel<T, KIND, REMAKE>;
    k<<<grid_of(a8->rows * per), kThreads, 0, s>>>(
        dy, lddy, a8->data, a8->scale, b8->data, b8->scale, a8->rows, (uint32_t)a8->cols, per, vec,
        da, ldda, db, lddb, REMAKE ? y8->data : nullptr, REMAKE ? y8->scale : nullptr);
    return cudaGetLastError() == cudaSuccess ? ARK_OK : ARK_E_CUDA;
}

bool same_shape(const ark_act8* a, const ark_act8* b) {
    return a->rows == b->rows && a->cols == b->cols && a->kind == b->kind;
}

}  // namespace
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
    if (!dy || !da || !db) return ARK_E_INVALID_ARG;
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
