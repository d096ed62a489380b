// Residual addition, RMS norm and an 8-bit output in one pass over a row (sm_100a).
//
//   h = round_s(x + residual)                    the updated residual stream, stored in the residual's type
//   y = round_x(h * rstd * weight)               rstd = 1/sqrt(mean(h^2) + eps), of the stored h, in fp32
//   MXFP8:          quantize_mxfp8(y)            32-element blocks, E8M0 scales in the 128x4 tiled layout
//   per-tensor FP8: quantize_per_tensor_fp8(y)   one device scalar
//
// The quantizers see y as the norm kernel would have stored it, so the packed output is that of the three
// separate operators, while h is written once and y never (unless it is asked for).
//
// Bound by HBM: 2 (x) + 2 (residual) + 2 (h) + 1.03 (codes, scales) bytes per 16-bit element.  One CTA takes a row and
// keeps it in registers between the two passes (a thread owns kChunks chunks of 16 elements, two lanes a block), so
// the only wait is the block-wide sum; rows too wide for that, or not aligned for 256-bit accesses, loop and read h
// back from where the same thread has just written it.
#include "ck_common.cuh"

namespace ck {
namespace {

struct AddNormArgs {
    const void* x;
    const void* residual;
    const void* weight;       // [D] in x's type, may be null
    const float* scale;       // per-tensor FP8 only
    void* sum;                // [N, D] contiguous in the residual's type (may be the residual itself)
    void* norm;               // [N, D] in x's type, may be null
    uint8_t* q;               // [N, D]
    uint8_t* sf;              // MXFP8: tiled block scales
    int64_t N, D;
    int64_t x_stride, res_stride;   // elements between rows
    int64_t sf_cpad;
    float eps;
    int e5m2;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the CTA, the same value in every thread (fixed order: warps' sums in turn).
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float s_part[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    v = warp_sum(v);
    if (lane == 0) s_part[warp] = v;
    __syncthreads();
    return warp_sum(lane < warps ? s_part[lane] : 0.0f);
}

// 16 elements, one 256-bit access per 16-bit chunk; not through the read-only path, since `sum` may be the
// residual's own memory.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, Raw16<T>& r) {
    constexpr int kWords = (int)(sizeof(r.w) / 4);
#pragma unroll
    for (int i = 0; i < kWords; i += 8)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]), "=r"(r.w[i + 4]), "=r"(r.w[i + 5]),
                       "=r"(r.w[i + 6]), "=r"(r.w[i + 7])
                     : "l"(reinterpret_cast<const uint32_t*>(p) + i) : "memory");
}

// The guarded form of the loads and stores: element by element, zeros beyond the row's end.
template <typename T>
__device__ __forceinline__ void load_guarded(const T* p, int64_t col, int64_t D, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = col + i < D ? Elem<T>::to_f32(p[col + i]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_guarded(T* p, int64_t col, int64_t D, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (col + i < D) p[col + i] = Elem<T>::from_f32(v[i]);
}

// y in x's type -> codes (and the scale byte) of the chunk.  All 32 lanes take part; `chunk` may lie behind the row's
// end (y is zero there).
template <typename T, bool kMx, bool kVec>
__device__ __forceinline__ void encode_chunk(const AddNormArgs& a, int64_t row, int64_t chunk, int lane, float inv, const float (&y)[16]) {
    const int64_t col = chunk * 16;
    uint2 p0, p1;
    if (kMx) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(y[j]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        float lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { lo[j] = y[j]; hi[j] = y[8 + j]; }
        uint32_t e;
        p0 = mxfp8_encode8(lo, amax, e);
        p1 = mxfp8_encode8(hi, amax, e);
        // eight lanes hold four blocks: their scale bytes are one word of the tile (zeros behind the row's end)
        uint32_t word = (lane & 1) ? 0u : e << (8 * ((lane >> 1) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        if ((lane & 7) == 0 && (chunk >> 1) < a.sf_cpad)
            *reinterpret_cast<uint32_t*>(a.sf + sf_offset(row, chunk >> 1, a.sf_cpad)) = word;
    } else {
        const float most = a.e5m2 ? 57344.0f : 448.0f;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = fminf(fmaxf(Elem<T>::round(__fmul_rn(y[4 * j + k], inv)), -most), most);
            w[j] = a.e5m2 ? cvt_e5m2x2(t[1], t[0]) | (cvt_e5m2x2(t[3], t[2]) << 16) : cvt_e4m3x2(t[1], t[0]) | (cvt_e4m3x2(t[3], t[2]) << 16);
        }
        p0 = make_uint2(w[0], w[1]);
        p1 = make_uint2(w[2], w[3]);
    }
    uint8_t* q = a.q + row * a.D + col;
    if (kVec) {
        if (col < a.D) *reinterpret_cast<uint4*>(q) = make_uint4(p0.x, p0.y, p1.x, p1.y);
    } else {
        const uint32_t w[4] = {p0.x, p0.y, p1.x, p1.y};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (col + i < a.D) q[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}

// kChunks > 0: the row fits kChunks chunks per thread and stays in registers; 0: any width.
template <typename T, typename S, bool kMx, int kChunks, bool kVec>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const AddNormArgs a) {
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 31;
    if (row >= a.N) {   // a padding row of the tiled scale buffer
        for (int64_t c4 = threadIdx.x; c4 < (a.sf_cpad >> 2); c4 += blockDim.x)
            *reinterpret_cast<uint32_t*>(a.sf + sf_offset(row, c4 * 4, a.sf_cpad)) = 0u;
        return;
    }
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const S* res = static_cast<const S*>(a.residual) + row * a.res_stride;
    const T* weight = static_cast<const T*>(a.weight);
    S* sum = static_cast<S*>(a.sum) + row * a.D;
    T* norm = a.norm ? static_cast<T*>(a.norm) + row * a.D : nullptr;
    const float inv = kMx ? 0.0f : Elem<T>::round(__fdiv_rn(1.0f, __ldg(a.scale)));
    const int64_t D = a.D, steps = ceil_div(D, (int64_t)16 * blockDim.x);   // every thread makes every step
    constexpr int kKept = kChunks > 0 ? kChunks : 1;
    float h[kKept][16];
    float ss = 0.0f;

    if (kChunks > 0) {
        Raw16<T> rx[kKept];
        Raw16<S> rr[kKept];
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
            const int64_t col = ((int64_t)i * blockDim.x + threadIdx.x) * 16;
            if (col < D) { load_chunk<T>(x + col, rx[i]); load_chunk<S>(res + col, rr[i]); }
            else { zero_raw16<T>(rx[i]); zero_raw16<S>(rr[i]); }
        }
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
            const int64_t col = ((int64_t)i * blockDim.x + threadIdx.x) * 16;
            float b[16];
            unpack16(rx[i], h[i]);
            unpack16(rr[i], b);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                h[i][j] = Elem<S>::round(__fadd_rn(h[i][j], b[j]));
                ss = fmaf(h[i][j], h[i][j], ss);
            }
            if (col < D) store16<S>(sum + col, h[i]);
        }
    } else {
        for (int64_t i = 0; i < steps; ++i) {
            const int64_t col = (i * blockDim.x + threadIdx.x) * 16;
            if (col >= D) continue;
            float b[16];
            if (kVec) {
                Raw16<T> rx;
                Raw16<S> rr;
                load_chunk<T>(x + col, rx);
                load_chunk<S>(res + col, rr);
                unpack16(rx, h[0]);
                unpack16(rr, b);
            } else {
                load_guarded<T>(x, col, D, h[0]);
                load_guarded<S>(res, col, D, b);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                h[0][j] = Elem<S>::round(__fadd_rn(h[0][j], b[j]));
                ss = fmaf(h[0][j], h[0][j], ss);
            }
            if (kVec) store16<S>(sum + col, h[0]);
            else store_guarded<S>(sum, col, D, h[0]);
        }
    }
    const float rstd = rsqrtf(block_sum(ss) / (float)D + a.eps);

    auto finish = [&](int64_t chunk, float (&v)[16]) {
        const int64_t col = chunk * 16;
        float w[16], y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = 1.0f;
        if (weight && col < D) {
            if (kVec) load16<T>(weight + col, w);
            else load_guarded<T>(weight, col, D, w);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = __fmul_rn(__fmul_rn(v[j], rstd), w[j]);
#pragma unroll
        for (int j = 0; j < 16; j += 2) Elem<T>::round2(y[j], y[j + 1]);
        if (col >= D) {
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = 0.0f;   // (a row of infinities: 0 * rstd is no number there)
        } else if (norm) {
            if (kVec) store16<T>(norm + col, y);
            else store_guarded<T>(norm, col, D, y);
        }
        encode_chunk<T, kMx, kVec>(a, row, chunk, lane, inv, y);
    };
    if (kChunks > 0) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) finish((int64_t)i * blockDim.x + threadIdx.x, h[i]);
    } else {
        for (int64_t i = 0; i < steps; ++i) {
            const int64_t chunk = i * blockDim.x + threadIdx.x, col = chunk * 16;
            if (!kVec || col >= D) load_guarded<S>(sum, col, D, h[0]);
            else {
                Raw16<S> r;
                load_chunk<S>(sum + col, r);
                unpack16(r, h[0]);
            }
            finish(chunk, h[0]);
        }
    }
}

template <typename T, typename S, bool kMx>
int launch(const AddNormArgs& a, bool vec, cudaStream_t stream) {
    // MXFP8 rows cover the scale columns' padding, too: 8 chunks per word of scale bytes
    const int64_t chunks = kMx ? a.sf_cpad * 2 : ceil_div(a.D, 16);
    const int64_t rows = kMx ? round_up(a.N, 128) : a.N;
    if (rows > 0x7fffffff) CK_FAIL(CK_ERR_SHAPE, "add_rmsnorm_quantize: %lld rows are too many", (long long)a.N);
    const int per = chunks <= 256 ? 1 : chunks <= 1024 ? 2 : 4;
    const int64_t want = round_up(ceil_div(chunks, per), 32);
    const unsigned threads = (unsigned)(want > 1024 ? 1024 : want);
    const unsigned grid = (unsigned)rows;
    if (!vec) add_rmsnorm_kernel<T, S, kMx, 0, false><<<grid, threads, 0, stream>>>(a);
    else if (want > 1024) add_rmsnorm_kernel<T, S, kMx, 0, true><<<grid, threads, 0, stream>>>(a);
    else if (per == 1) add_rmsnorm_kernel<T, S, kMx, 1, true><<<grid, threads, 0, stream>>>(a);
    else if (per == 2) add_rmsnorm_kernel<T, S, kMx, 2, true><<<grid, threads, 0, stream>>>(a);
    else add_rmsnorm_kernel<T, S, kMx, 4, true><<<grid, threads, 0, stream>>>(a);
    return launch_status("add_rmsnorm_quantize");
}

template <typename T, typename S>
int launch_fmt(const AddNormArgs& a, bool mx, bool vec, cudaStream_t stream) {
    return mx ? launch<T, S, true>(a, vec, stream) : launch<T, S, false>(a, vec, stream);
}

}  // namespace
}  // namespace ck

extern "C" int launch_add_rmsnorm_quantize_kernel(const void* x, const void* residual, const void* weight, const void* scale,
                                                  void* sum_out, void* norm_out, void* output, void* block_scales, int64_t N,
                                                  int64_t D, int64_t x_row_stride, int64_t residual_row_stride, float eps,
                                                  int dtype_code, int residual_dtype_code, int output_dtype_code,
                                                  cudaStream_t stream) {
    using namespace ck;
    const bool mx = block_scales != nullptr;
    if (!x || !residual || !sum_out || !output || (!mx && !scale)) CK_FAIL(CK_ERR_NULL, "add_rmsnorm_quantize: null pointer");
    if (mx && output_dtype_code != CK_E4M3) CK_FAIL(CK_ERR_DTYPE, "add_rmsnorm_quantize: MXFP8 data is E4M3");
    if (output_dtype_code != CK_E4M3 && output_dtype_code != CK_E5M2)
        CK_FAIL(CK_ERR_DTYPE, "add_rmsnorm_quantize: output dtype code %d (E4M3 or E5M2)", output_dtype_code);
    if (dtype_code != CK_F32 && dtype_code != CK_F16 && dtype_code != CK_BF16)
        CK_FAIL(CK_ERR_DTYPE, "add_rmsnorm_quantize: dtype code %d", dtype_code);
    if (residual_dtype_code != dtype_code && residual_dtype_code != CK_F32)
        CK_FAIL(CK_ERR_DTYPE, "add_rmsnorm_quantize: the residual has x's dtype or fp32");
    if (N <= 0 || D <= 0 || x_row_stride < D || residual_row_stride < D || (mx && D % 32 != 0))
        CK_FAIL(CK_ERR_SHAPE, "add_rmsnorm_quantize: bad shape N=%lld D=%lld (MXFP8: D a multiple of 32)", (long long)N, (long long)D);
    if (sum_out == residual && residual_row_stride != D)
        CK_FAIL(CK_ERR_SHAPE, "add_rmsnorm_quantize: a residual updated in place is contiguous");
    if (mx && (reinterpret_cast<uintptr_t>(block_scales) & 3)) CK_FAIL(CK_ERR_ALIGN, "add_rmsnorm_quantize: block scales must be 4-byte aligned");
    const int64_t es = dtype_code == CK_F32 ? 4 : 2, rs = residual_dtype_code == CK_F32 ? 4 : 2;
    const bool vec = D % 16 == 0 && aligned32(x) && aligned32(residual) && aligned32(sum_out) && (!norm_out || aligned32(norm_out)) &&
                     (!weight || aligned32(weight)) && aligned16(output) && (x_row_stride * es) % 32 == 0 &&
                     (residual_row_stride * rs) % 32 == 0;
    AddNormArgs a{x, residual, weight, static_cast<const float*>(scale), sum_out, norm_out, static_cast<uint8_t*>(output),
                  static_cast<uint8_t*>(block_scales), N, D, x_row_stride, residual_row_stride, mx ? round_up(D / 32, 4) : 0, eps,
                  output_dtype_code == CK_E5M2};
    if (dtype_code == CK_F32) return launch_fmt<float, float>(a, mx, vec, stream);
    if (dtype_code == CK_F16)
        return residual_dtype_code == CK_F32 ? launch_fmt<__half, float>(a, mx, vec, stream) : launch_fmt<__half, __half>(a, mx, vec, stream);
    return residual_dtype_code == CK_F32 ? launch_fmt<__nv_bfloat16, float>(a, mx, vec, stream)
                                         : launch_fmt<__nv_bfloat16, __nv_bfloat16>(a, mx, vec, stream);
}
