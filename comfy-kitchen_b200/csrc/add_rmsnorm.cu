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
//
// Measured: 16384 x 8192 bf16 to MXFP8 in 152.8 us back to back (6.18 TB/s, 96 % of the copy rate; 141 in a short burst),
// 4608 x 8192 bf16 with an fp32 residual to per-tensor FP8 in 68.2 us (6.09 TB/s, 94 %), one row of 4096 in 2.1 us of a graph.  The MXFP8
// form has instructions to spare only since pairs are worked on together (add, squares, products, maximum) and the
// scale needs no division: 28.5 instructions an element took 74 % of the issue slots and 164 us, 21 take 58 %.
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

// y (fp32) rounded to x's type, as it is stored and as fp32 again, and the largest magnitude (NaN not counted).
// 16-bit types keep the pairs packed: one conversion, one maximum for two elements.
template <typename T> struct Rounded;
template <> struct Rounded<float> {
    float v[16];
    __device__ void set(int i, float2 p) { v[2 * i] = p.x; v[2 * i + 1] = p.y; }
    __device__ float2 get(int i) const { return make_float2(v[2 * i], v[2 * i + 1]); }
    __device__ float amax() const {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
        return m;
    }
    __device__ void store(float* p) const { store16<float>(p, v); }
};
template <> struct Rounded<__nv_bfloat16> {
    uint32_t w[8];
    __device__ void set(int i, float2 p) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ float2 get(int i) const { return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)); }
    __device__ float amax() const {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("max.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
        return fmaxf(__uint_as_float((m << 16) & 0x7fffffffu), __uint_as_float(m & 0x7fff0000u));
    }
    __device__ void store(__nv_bfloat16* p) const { stg256(p, w); }
};
template <> struct Rounded<__half> {
    uint32_t w[8];
    __device__ void set(int i, float2 p) {
        const __half2 h = __floats2half2_rn(p.x, p.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ float2 get(int i) const { return __half22float2(*reinterpret_cast<const __half2*>(&w[i])); }
    __device__ float amax() const {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("max.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
        m &= 0x7fff7fffu;
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
        return fmaxf(f.x, f.y);
    }
    __device__ void store(__half* p) const { stg256(p, w); }
};

// y -> codes (and the scale byte) of the chunk.  All 32 lanes take part; `chunk` may lie behind the row's end (y is
// zero there).
//
// MXFP8's scale is the smallest power of two not below amax / 448.  448 = 1.75 x 2^8, and no fp32 quotient by it rounds down
// to a power of two (the float behind 1.75 x 2^k is 0.57 units of the quotient's last place away), so away from the ends of
// the range the exponent comes from amax's own bits, without a division; there the general form serves.
template <typename T, bool kMx, bool kVec>
__device__ __forceinline__ void encode_chunk(const AddNormArgs& a, int64_t row, int64_t sf_row, int64_t chunk, int lane, float inv,
                                             const Rounded<T>& y) {
    const int64_t col = chunk * 16;
    uint32_t w[4];
    if (kMx) {
        float amax = y.amax();
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        const uint32_t bits = __float_as_uint(amax);
        uint32_t e = (bits + 0x1fffffu) >> 23;   // + 8
        if (bits < 0x7f800000u && e >= 10u) {
            e -= 8u;
            const float up = __uint_as_float((254u - e) << 23);   // 2^(127 - e)
            const float2 up2 = make_float2(up, up);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __fmul2_rn(y.get(2 * j), up2), g = __fmul2_rn(y.get(2 * j + 1), up2);
                w[j] = cvt_e4m3x2(f.y, f.x) | (cvt_e4m3x2(g.y, g.x) << 16);
            }
        } else {
            float lo[8], hi[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = y.get(j), g = y.get(4 + j);
                lo[2 * j] = f.x; lo[2 * j + 1] = f.y;
                hi[2 * j] = g.x; hi[2 * j + 1] = g.y;
            }
            const uint2 p0 = mxfp8_encode8(lo, amax, e), p1 = mxfp8_encode8(hi, amax, e);
            w[0] = p0.x; w[1] = p0.y; w[2] = p1.x; w[3] = p1.y;
        }
        // eight lanes hold four blocks: their scale bytes are one word of the tile (zeros behind the row's end)
        uint32_t word = e << (4 * (lane & 6));   // lanes 2 i and 2 i + 1 hold byte i twice
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        if ((lane & 7) == 0 && (chunk >> 1) < a.sf_cpad) *reinterpret_cast<uint32_t*>(a.sf + sf_row + (chunk >> 3) * 512) = word;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // (the conversions saturate; NaN stays NaN)
            float t[4];
            const float2 f = y.get(2 * j), g = y.get(2 * j + 1);
            t[0] = __fmul_rn(f.x, inv); t[1] = __fmul_rn(f.y, inv); t[2] = __fmul_rn(g.x, inv); t[3] = __fmul_rn(g.y, inv);
            Elem<T>::round2(t[0], t[1]);
            Elem<T>::round2(t[2], t[3]);
            w[j] = a.e5m2 ? cvt_e5m2x2(t[1], t[0]) | (cvt_e5m2x2(t[3], t[2]) << 16) : cvt_e4m3x2(t[1], t[0]) | (cvt_e4m3x2(t[3], t[2]) << 16);
        }
    }
    uint8_t* q = a.q + row * a.D + col;
    if (kVec) {
        if (col < a.D) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (col + i < a.D) q[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}

// h = round_s(x + residual) and the sum of its squares, two elements an instruction.
template <typename S>
__device__ __forceinline__ void add_residual(float (&h)[16], const float (&b)[16], float2& ss) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        float2 t = __fadd2_rn(make_float2(h[j], h[j + 1]), make_float2(b[j], b[j + 1]));
        Elem<S>::round2(t.x, t.y);
        ss = __ffma2_rn(t, t, ss);
        h[j] = t.x; h[j + 1] = t.y;
    }
}

// kChunks > 0: the row fits kChunks chunks per thread and stays in registers; 0: any width.
template <typename T, typename S, bool kMx, int kChunks, bool kVec>
__global__ void __launch_bounds__(kChunks == 0 ? 1024 : kChunks == 1 ? 256 : 512, kChunks == 1 ? 4 : kChunks == 2 ? 2 : 1)
add_rmsnorm_kernel(const AddNormArgs a) {
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
    const int64_t sf_row = kMx ? sf_offset(row, 0, a.sf_cpad) : 0;
    const int64_t D = a.D, steps = ceil_div(D, (int64_t)16 * blockDim.x);   // every thread makes every step
    constexpr int kKept = kChunks > 0 ? kChunks : 1;
    float h[kKept][16];
    float2 ss = make_float2(0.0f, 0.0f);

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
            add_residual<S>(h[i], b, ss);
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
            add_residual<S>(h[0], b, ss);
            if (kVec) store16<S>(sum + col, h[0]);
            else store_guarded<S>(sum, col, D, h[0]);
        }
    }
    const float rstd = rsqrtf(block_sum(ss.x + ss.y) / (float)D + a.eps);

    auto finish = [&](int64_t chunk, float (&v)[16]) {
        const int64_t col = chunk * 16;
        float w[16];
        if (weight && col < D) {
            if (kVec) load16<T>(weight + col, w);
            else load_guarded<T>(weight, col, D, w);
        }
        Rounded<T> y;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float2 t = __fmul2_rn(make_float2(v[2 * j], v[2 * j + 1]), make_float2(rstd, rstd));
            if (weight) t = __fmul2_rn(t, make_float2(w[2 * j], w[2 * j + 1]));
            if (col >= D) t = make_float2(0.0f, 0.0f);   // (a row of infinities: 0 * rstd is no number there)
            y.set(j, t);
        }
        if (norm && col < D) {
            if (kVec) y.store(norm + col);
            else {
                float t[16];
#pragma unroll
                for (int j = 0; j < 8; ++j) { t[2 * j] = y.get(j).x; t[2 * j + 1] = y.get(j).y; }
                store_guarded<T>(norm, col, D, t);
            }
        }
        encode_chunk<T, kMx, kVec>(a, row, sf_row, chunk, lane, inv, y);
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
    const bool kept = vec && want <= 512;
    const unsigned threads = (unsigned)(kept || want <= 1024 ? want : 1024);
    const unsigned grid = (unsigned)rows;
    if (!vec) add_rmsnorm_kernel<T, S, kMx, 0, false><<<grid, threads, 0, stream>>>(a);
    else if (!kept) add_rmsnorm_kernel<T, S, kMx, 0, true><<<grid, threads, 0, stream>>>(a);
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
    // An element is read and written by the same thread, so an output may have x's or the residual's place, but no other.
    const int64_t wide = mx ? round_up(D / 32, 4) : 0;
    const Memory in[4] = {{x, N, x_row_stride * es, D * es}, {residual, N, residual_row_stride * rs, D * rs}, memory_of(weight, D * es), memory_of(scale, 4)};
    const Memory out[4] = {{sum_out, N, D * rs, D * rs}, {norm_out, N, D * es, D * es}, memory_of(output, N * D), memory_of(block_scales, round_up(N, 128) * wide)};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < 4; ++j)
            if (overlap(out[i], in[j]) && !(j < 2 && same_place(out[i], in[j])))
                CK_FAIL(CK_ERR_UNSUPPORTED, "add_rmsnorm_quantize: an output overlaps an input and has not its place");
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) CK_FAIL(CK_ERR_UNSUPPORTED, "add_rmsnorm_quantize: two outputs overlap");
    }
    const bool vec = D % 16 == 0 && aligned32(x) && aligned32(residual) && aligned32(sum_out) && (!norm_out || aligned32(norm_out)) &&
                     (!weight || aligned32(weight)) && aligned16(output) && (x_row_stride * es) % 32 == 0 &&
                     (residual_row_stride * rs) % 32 == 0;
    AddNormArgs a{x, residual, weight, static_cast<const float*>(scale), sum_out, norm_out, static_cast<uint8_t*>(output),
                  static_cast<uint8_t*>(block_scales), N, D, x_row_stride, residual_row_stride, wide, eps,
                  output_dtype_code == CK_E5M2};
    if (dtype_code == CK_F32) return launch_fmt<float, float>(a, mx, vec, stream);
    if (dtype_code == CK_F16)
        return residual_dtype_code == CK_F32 ? launch_fmt<__half, float>(a, mx, vec, stream) : launch_fmt<__half, __half>(a, mx, vec, stream);
    return residual_dtype_code == CK_F32 ? launch_fmt<__nv_bfloat16, float>(a, mx, vec, stream)
                                         : launch_fmt<__nv_bfloat16, __nv_bfloat16>(a, mx, vec, stream);
}
