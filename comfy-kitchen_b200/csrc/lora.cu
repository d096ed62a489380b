// Low-rank adapters of many requests beside a shared projection (sm_100a).
//
//   out[t] = y[t] + scale[a] * B_a (A_a x[t]),   a = ids[t];  out[t] = y[t] where a is no adapter (outside [0, L))
//
// y is the shared projection's output for the row, A_a [R, K], B_a [N, R].  Sums in fp32, one rounding at the end.
#include "ck_common.cuh"

namespace ck {
namespace {

constexpr int kMaxRank = 256;

struct LoraArgs {
    const void* y;
    const void* x;
    const void* a;          // [L, R, K]
    const void* b;          // [L, N, R]
    const void* ids;        // int32 or int64, one per rows_per_id rows
    const float* scales;    // [L] or null
    void* out;
    int64_t rows, K, N, R, L;
    int64_t y_stride, x_stride, out_stride;
    int64_t rows_per_id;
    int ids64;
};

__device__ __forceinline__ int adapter_of(const LoraArgs& p, int64_t row) {
    const int64_t i = row / p.rows_per_id;
    const int64_t id = p.ids64 ? (int64_t)__ldg(static_cast<const long long*>(p.ids) + i) : (int64_t)__ldg(static_cast<const int*>(p.ids) + i);
    return id < 0 || id >= p.L ? -1 : (int)id;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One row per CTA: a warp takes one row of A at a time, then every thread one column of the output.
template <typename T>
__global__ void __launch_bounds__(256) lora_row_kernel(const LoraArgs p) {
    __shared__ float s_low[kMaxRank];
    const int64_t row = blockIdx.x;
    const int id = adapter_of(p, row);
    const T* y = static_cast<const T*>(p.y) + row * p.y_stride;
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    if (id < 0) {
        if (p.out != p.y)
            for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) out[n] = y[n];
        return;
    }
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* a = static_cast<const T*>(p.a) + (int64_t)id * p.R * p.K;
    const T* b = static_cast<const T*>(p.b) + (int64_t)id * p.N * p.R;
    const float scale = p.scales ? __ldg(p.scales + id) : 1.0f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < p.R; r += blockDim.x >> 5) {
        float sum = 0.0f;
        for (int64_t k = lane * 8; k < p.K; k += 256) {
            float u[8], v[8];
            load8<T>(x + k, u);
            load8<T>(a + r * p.K + k, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(u[j], v[j], sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) s_low[r] = sum;
    }
    __syncthreads();
    for (int64_t n = threadIdx.x; n < p.N; n += blockDim.x) {
        float sum = 0.0f;
        for (int r = 0; r < p.R; r += 8) {
            float v[8];
            load8<T>(b + n * p.R + r, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(s_low[r + j], v[j], sum);
        }
        out[n] = Elem<T>::from_f32(fmaf(scale, sum, Elem<T>::to_f32(y[n])));
    }
}

}  // namespace
}  // namespace ck

extern "C" int launch_lora_add_kernel(const void* y, const void* x, const void* a, const void* b, const void* ids,
                                      const float* scales, void* out, int64_t rows, int64_t K, int64_t N, int64_t rank,
                                      int64_t adapters, int64_t y_row_stride, int64_t x_row_stride, int64_t out_row_stride,
                                      int64_t rows_per_id, int dtype_code, bool ids_64bit, cudaStream_t stream) {
    using namespace ck;
    if (!y || !x || !a || !b || !ids || !out) CK_FAIL(CK_ERR_NULL, "lora_add: null pointer");
    if (dtype_code != CK_F16 && dtype_code != CK_BF16) CK_FAIL(CK_ERR_DTYPE, "lora_add: dtype code %d (bf16 or fp16)", dtype_code);
    if (rows <= 0 || rows > 0x7fffffff || K <= 0 || K > 0x7fffffff || N <= 0 || N > 0x7fffffff || adapters <= 0 || adapters > 0x7fffffff ||
        K % 8 != 0 || N % 8 != 0 || rows_per_id <= 0 || x_row_stride < K || y_row_stride < N || out_row_stride < N)
        CK_FAIL(CK_ERR_SHAPE, "lora_add: bad shape rows=%lld K=%lld N=%lld adapters=%lld (K and N multiples of 8)", (long long)rows,
                (long long)K, (long long)N, (long long)adapters);
    if (rank <= 0 || rank % 8 != 0 || rank > kMaxRank) CK_FAIL(CK_ERR_SHAPE, "lora_add: rank %lld (a multiple of 8, at most %d)", (long long)rank, kMaxRank);
    if (!aligned16(y) || !aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(out) || ((x_row_stride | y_row_stride | out_row_stride) & 7))
        CK_FAIL(CK_ERR_ALIGN, "lora_add: tensors and row strides must be 16-byte aligned");
    const LoraArgs p{y, x, a, b, ids, scales, out, rows, K, N, rank, adapters, y_row_stride, x_row_stride, out_row_stride, rows_per_id, ids_64bit};
    if (dtype_code == CK_BF16) lora_row_kernel<__nv_bfloat16><<<(unsigned)rows, 256, 0, stream>>>(p);
    else lora_row_kernel<__half><<<(unsigned)rows, 256, 0, stream>>>(p);
    return launch_status("lora_add");
}
