// Low-rank adapters of many requests beside a shared projection (sm_100a).
//
//   out[t] = y[t] + scale[a] * B_a (A_a x[t]),   a = ids[t];  out[t] = y[t] where a is no adapter (outside [0, L))
//
// y [T, N] is the shared projection's output for the rows x [T, K]; A_a [R, K], B_a [N, R].
//
// Bound by HBM in either direction: x is read once, y read and out written once (2 K + 4 N bytes a row), each used adapter
// once; the products' 2 R (K + N) flop a row stay below that up to a rank of about 128.  Two forms:
//   few rows:   one CTA per row.
//   many rows:  two kernels of 128-row tiles on the tensor cores (tcgen05), joined by the low-rank vectors in fp32.
//               shrink:  low[t, :] = A x[t], the K axis split over CTAs (each split writes its own partial sums, which
//                        the next kernel adds in order: no atomics, the same bits every time);
//               expand:  out = y + scale * (B low), y tiles fetched and out tiles stored by TMA while the products run.
// Ids are looked at on the device: a tile lists the adapters that its rows ask for, computes each one's product for all 128
// rows and keeps a row's own (a row of another request never enters a sum, whatever it holds).  Requests that lie behind
// one another cost nothing extra; a tile of 128 different adapters reads 128 adapters, as it must.
//
// Rounding: sums in fp32.  The low-rank vector is the second product's 16-bit operand: it goes in as two parts, the
// rounded value and what the rounding left (for fp16 scaled by a power of two per row, which keeps large and small vectors
// in range), so that about 16 bits (fp16: 22) of it are used and the output's rounding is the only one that shows.
#include "ck_common.cuh"
#include "ck_tc.cuh"

namespace ck {
namespace {

constexpr int kMaxRank = 256;
constexpr int kTile = 128;          // rows of a tile (the MMA's M)
constexpr int kThreads = 192;       // warp 0: TMA, warp 1: MMA, warps 2-5: epilogue, one per 32 rows of the tile
constexpr int kTileBytes = kTile * 128;   // 128 rows x 64 elements
constexpr int kSmemMost = 232448;

constexpr int kShrinkColumns = 256;   // two accumulators of up to 128 columns, or one of up to 256; two CTAs share an SM's TMEM

__device__ int g_lora_status = 0;
enum : int { kWaitFull = 1, kWaitEmpty = 2, kWaitAcc = 3, kWaitAccFree = 4, kWaitLow = 5, kWaitY = 6, kWaitYFree = 7, kWaitDrain = 8 };

struct LoraArgs {
    const void* y;
    const void* x;
    const void* a;          // [L, R, K]
    const void* b;          // [L, N, R]
    const void* ids;        // int32 or int64, one per rows_per_id rows
    const float* scales;    // [L] or null
    void* out;
    float* low;             // [splits, rows, R] (many rows)
    int64_t rows, K, N, R, L;
    int64_t y_stride, x_stride, out_stride;
    int64_t rows_per_id;
    int ids64;
    int splits;
};

__device__ __forceinline__ int adapter_of(const LoraArgs& p, int64_t row) {
    const int64_t i = p.rows_per_id == 1 ? row : row / p.rows_per_id;
    const int64_t id = p.ids64 ? (int64_t)__ldg(static_cast<const long long*>(p.ids) + i) : (int64_t)__ldg(static_cast<const int*>(p.ids) + i);
    return id < 0 || id >= p.L ? -1 : (int)id;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ------------------------------------------------------------------ few rows

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

// ------------------------------------------------------------------ many rows

// The adapters that the tile's rows ask for, in the order of their first rows: their number, which of them row
// 32 * quarter + lane asks for (mine, -1: none) and, where `list` is given, their ids.  By a whole warp.
__device__ __forceinline__ int tile_adapters(const LoraArgs& p, int64_t row0, int lane, int quarter, int& mine, int* list) {
    int id[4];
    uint32_t left[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t row = row0 + 32 * q + lane;
        id[q] = row < p.rows ? adapter_of(p, row) : -1;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) left[q] = __ballot_sync(0xffffffffu, id[q] >= 0);
    mine = -1;
    int count = 0;
    while (left[0] | left[1] | left[2] | left[3]) {
        int cur = -1;
#pragma unroll
        for (int q = 3; q >= 0; --q) {   // (the first quarter that has rows left decides)
            const int first = __shfl_sync(0xffffffffu, id[q], left[q] ? __ffs(left[q]) - 1 : 0);
            if (left[q]) cur = first;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            left[q] &= ~__ballot_sync(0xffffffffu, id[q] == cur);
            if (q == quarter && id[q] == cur) mine = count;
        }
        if (list && lane == 0) list[count] = cur;
        ++count;
    }
    __syncwarp();
    return count;
}

struct ShrinkPlan {
    int splits, groups;         // K parts; adapters of a tile are dealt to `groups` CTAs
    int k_tiles, rn;            // 64-element steps of K; R rounded up to 16 (the MMA's N)
    int stages, accs;           // ring of operand tiles; accumulators in TMEM
    int smem;
};

// low[split][t][:] = A_{ids[t]} x[t] over this CTA's part of K.
__global__ void __launch_bounds__(kThreads)
lora_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const LoraArgs p,
                   const ShrinkPlan plan, const bool bf16) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stage_bytes = kTileBytes + plan.rn * 128;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + plan.stages * stage_bytes);
    uint64_t* empty = full + plan.stages;
    uint64_t* acc_full = empty + plan.stages;     // [2]
    uint64_t* acc_empty = acc_full + 2;           // [2]
    uint64_t* drain = acc_empty + 2;
    int* s_list = reinterpret_cast<int*>(drain + 1);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_list + kTile);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row0 = (int64_t)blockIdx.x * kTile;
    const int split = blockIdx.y, group = blockIdx.z;
    int mine;
    const int count = tile_adapters(p, row0, lane, warp & 3, mine, warp == 0 ? s_list : nullptr);
    if (group >= count) return;   // (the same for every warp)
    const int k0 = (int)((int64_t)plan.k_tiles * split / plan.splits), k1 = (int)((int64_t)plan.k_tiles * (split + 1) / plan.splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.stages; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 4); }
        tc::mbar_init(drain, 1);
        *s_abort = 0;
        tc::mbar_init_done();
    }
    if (warp == 1) tc::tmem_alloc(s_tmem, kShrinkColumns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int j = group; j < count && ok; j += plan.groups) {
            const int id = s_list[j];
            for (int kt = k0; kt < k1; ++kt, ++it) {
                const int s = it % plan.stages;
                if (it >= (uint32_t)plan.stages) ok = tc::mbar_wait(&empty[s], (it / plan.stages - 1) & 1, s_abort, &g_lora_status, kWaitEmpty);
                if (!ok) break;
                if (lane == 0) {
                    uint8_t* st = smem + s * stage_bytes;
                    tc::mbar_expect_tx(&full[s], (uint32_t)stage_bytes);
                    tc::tma_load_2d(st, &map_x, kt * 64, (int)row0, &full[s]);
                    tc::tma_load_3d(st + kTileBytes, &map_a, kt * 64, 0, id, &full[s]);
                }
                __syncwarp();
            }
        }
        if (!ok)   // copies in flight land before the CTA leaves
            for (uint32_t i = it > (uint32_t)plan.stages ? it - plan.stages : 0; i < it; ++i)
                for (uint32_t n = 0; n < tc::kSpinLimit && !tc::mbar_try_wait(&full[i % plan.stages], (i / plan.stages) & 1); ++n) {}
    } else if (warp == 1) {
        const uint32_t id = tc::idesc(bf16, plan.rn);
        uint32_t it = 0, n = 0;
        bool ok = true;
        for (int j = group; j < count && ok; j += plan.groups, ++n) {
            const uint32_t buf = n % plan.accs;
            if (n >= (uint32_t)plan.accs) ok = tc::mbar_wait(&acc_empty[buf], (n / plan.accs - 1) & 1, s_abort, &g_lora_status, kWaitAccFree);
            if (!ok) break;
            tc::fence_after();
            for (int kt = k0; kt < k1; ++kt, ++it) {
                const int s = it % plan.stages;
                ok = tc::mbar_wait(&full[s], (it / plan.stages) & 1, s_abort, &g_lora_status, kWaitFull);
                if (!ok) break;
                tc::fence_after();
                const uint32_t da = tc::desc_lo(smem + s * stage_bytes), db = tc::desc_lo(smem + s * stage_bytes + kTileBytes);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma_16bit(tmem + buf * kTile, da + 2 * k, db + 2 * k, id, kt > k0 || k > 0);
                tc::commit(&empty[s]);
            }
            if (ok) tc::commit(&acc_full[buf]);
        }
        if (!ok) {   // MMAs in flight end before the operands and the TMEM go
            tc::commit(drain);
            for (uint32_t i = 0; i < tc::kSpinLimit && !tc::mbar_try_wait(drain, 0); ++i) {}
        }
    } else {
        const int64_t row = row0 + (warp & 3) * 32 + lane;
        float* low = p.low + ((int64_t)split * p.rows + row) * p.R;
        uint32_t n = 0;
        for (int j = group; j < count; j += plan.groups, ++n) {
            const uint32_t buf = n % plan.accs;
            if (!tc::mbar_wait(&acc_full[buf], (n / plan.accs) & 1, s_abort, &g_lora_status, kWaitAcc)) break;
            tc::fence_after();
            if (__any_sync(0xffffffffu, mine == j)) {
                for (int c = 0; c < plan.rn; c += 16) {
                    uint32_t v[16];
                    tc::ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * kTile + c, v);
                    tc::wait_ld();
                    if (mine == j) {
                        float4* dst = reinterpret_cast<float4*>(low + c);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (c + 4 * i < p.R)
                                dst[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    }
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, kShrinkColumns);
}

struct ExpandPlan {
    int64_t steps, items;       // column steps of a tile; tiles x steps
    int blocks;                 // 64-element blocks of R
    int b_stages, y_stages;
    int smem;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// The partial sums of 8 elements of a row's low-rank vector, added in the order of the splits.
__device__ __forceinline__ void low_sum8(const LoraArgs& p, int64_t row, int r, float (&v)[8]) {
    const float* src = p.low + row * p.R + r;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    for (int s = 0; s < p.splits; ++s, src += p.rows * p.R) {
        const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
}

// Writes this thread's row of the low-rank tile as two 16-bit operands (swizzled; hi, then lo) and returns the power of
// two that the products have to be multiplied by.
template <typename T>
__device__ __forceinline__ float put_low(const LoraArgs& p, const ExpandPlan& plan, uint8_t* s_low, int64_t row, int r_in_tile, bool has) {
    float down = 1.0f, up = 1.0f;
    if (sizeof(T) == 2 && Elem<T>::code == CK_F16 && has) {
        float most = 0.0f;
        for (int r = 0; r < p.R; r += 8) {
            float v[8];
            low_sum8(p, row, r, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
        }
        const int e = (int)(__float_as_uint(most) >> 23) - 127;   // most is in [2^e, 2^(e+1))
        if (e < 127 && e > -126) {                                // (not for zeros, infinities and what fp32 itself barely holds)
            up = __uint_as_float((uint32_t)(e + 127) << 23);
            down = __uint_as_float((uint32_t)(127 - e) << 23);
        }
    }
    const int padded = (int)round_up(p.R, 16);
    for (int r = 0; r < padded; r += 8) {
        float v[8];
        if (has && r < p.R) low_sum8(p, row, r, v);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[2 * i] * down, b = v[2 * i + 1] * down;
            float ha = Elem<T>::round(a), hb = Elem<T>::round(b);
            hi[i] = pack2<T>(ha, hb);
            lo[i] = pack2<T>(isfinite(ha) ? a - ha : 0.0f, isfinite(hb) ? b - hb : 0.0f);   // (an infinity stays one)
        }
        uint8_t* dst = s_low + (r >> 6) * kTileBytes + r_in_tile * 128 + ((((r & 63) >> 3) ^ (r_in_tile & 7)) << 4);
        *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + plan.blocks * kTileBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    return up;
}

// Persistent CTAs take equal runs of (tile, column step) items.  kN columns a step.
template <typename T, int kN>
__global__ void __launch_bounds__(kThreads, 1)
lora_expand_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_y,
                   const __grid_constant__ CUtensorMap map_out, const LoraArgs p, const ExpandPlan plan) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int kHalves = kN / 64;
    constexpr int kYBytes = kHalves * kTileBytes;
    const int b_bytes = plan.blocks * kN * 128;
    uint8_t* s_low = smem;                                             // hi blocks, lo blocks
    uint8_t* s_b = s_low + 2 * plan.blocks * kTileBytes;
    uint8_t* s_y = s_b + plan.b_stages * b_bytes;
    uint64_t* b_full = reinterpret_cast<uint64_t*>(s_y + plan.y_stages * kYBytes);
    uint64_t* b_empty = b_full + plan.b_stages;
    uint64_t* y_full = b_empty + plan.b_stages;
    uint64_t* y_empty = y_full + plan.y_stages;
    uint64_t* acc_full = y_empty + plan.y_stages;                      // [2]
    uint64_t* acc_empty = acc_full + 2;                                // [2]
    uint64_t* low_full = acc_empty + 2;
    uint64_t* drain = low_full + 1;
    int* s_list = reinterpret_cast<int*>(drain + 1);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_list + kTile);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = plan.items * blockIdx.x / gridDim.x, last = plan.items * (blockIdx.x + 1) / gridDim.x;
    const bool in_place = p.out == p.y;

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.b_stages; ++s) { tc::mbar_init(&b_full[s], 1); tc::mbar_init(&b_empty[s], 1); }
        for (int s = 0; s < plan.y_stages; ++s) { tc::mbar_init(&y_full[s], 1); tc::mbar_init(&y_empty[s], 4); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 4); }
        tc::mbar_init(low_full, 4);
        tc::mbar_init(drain, 1);
        *s_abort = 0;
        tc::mbar_init_done();
    }
    if (warp == 1) tc::tmem_alloc(s_tmem, 2 * kN);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp == 0) {
        uint32_t bi = 0, yi = 0;
        bool ok = true;
        for (int64_t item = first; item < last && ok;) {
            const int64_t tile = item / plan.steps, begin = item - tile * plan.steps, end = min(plan.steps, begin + last - item);
            item += end - begin;
            int mine;
            const int count = tile_adapters(p, tile * kTile, lane, 0, mine, s_list);
            if (count == 0 && in_place) continue;
            for (int64_t step = begin; step < end && ok; ++step) {
                {
                    const int s = yi % plan.y_stages;
                    if (yi >= (uint32_t)plan.y_stages) ok = tc::mbar_wait(&y_empty[s], (yi / plan.y_stages - 1) & 1, s_abort, &g_lora_status, kWaitYFree);
                    if (!ok) break;
                    if (lane == 0) {
                        tc::mbar_expect_tx(&y_full[s], kYBytes);
#pragma unroll
                        for (int h = 0; h < kHalves; ++h)
                            tc::tma_load_2d(s_y + s * kYBytes + h * kTileBytes, &map_y, (int)(step * kN + h * 64), (int)(tile * kTile), &y_full[s]);
                    }
                    ++yi;
                    __syncwarp();
                }
                for (int j = 0; j < count; ++j, ++bi) {
                    const int s = bi % plan.b_stages;
                    if (bi >= (uint32_t)plan.b_stages) ok = tc::mbar_wait(&b_empty[s], (bi / plan.b_stages - 1) & 1, s_abort, &g_lora_status, kWaitEmpty);
                    if (!ok) break;
                    if (lane == 0) {
                        tc::mbar_expect_tx(&b_full[s], (uint32_t)b_bytes);
                        for (int k = 0; k < plan.blocks; ++k)
                            tc::tma_load_3d(s_b + s * b_bytes + k * kN * 128, &map_b, k * 64, (int)(step * kN), s_list[j], &b_full[s]);
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok) {   // copies in flight land before the CTA leaves
            for (uint32_t i = bi > (uint32_t)plan.b_stages ? bi - plan.b_stages : 0; i < bi; ++i)
                for (uint32_t n = 0; n < tc::kSpinLimit && !tc::mbar_try_wait(&b_full[i % plan.b_stages], (i / plan.b_stages) & 1); ++n) {}
            for (uint32_t i = yi > (uint32_t)plan.y_stages ? yi - plan.y_stages : 0; i < yi; ++i)
                for (uint32_t n = 0; n < tc::kSpinLimit && !tc::mbar_try_wait(&y_full[i % plan.y_stages], (i / plan.y_stages) & 1); ++n) {}
        }
    } else if (warp == 1) {
        const uint32_t id = tc::idesc(Elem<T>::code == CK_BF16, kN);
        const int k_steps = (int)ceil_div(p.R, 16);
        uint32_t n = 0, seg = 0;
        bool ok = true;
        for (int64_t item = first; item < last && ok;) {
            const int64_t tile = item / plan.steps, begin = item - tile * plan.steps, end = min(plan.steps, begin + last - item);
            item += end - begin;
            int mine;
            const int count = tile_adapters(p, tile * kTile, lane, 0, mine, nullptr);
            if (count == 0) continue;
            ok = tc::mbar_wait(low_full, seg++ & 1, s_abort, &g_lora_status, kWaitLow);
            for (int64_t i = 0; i < (end - begin) * count && ok; ++i, ++n) {
                const uint32_t buf = n & 1;
                const int s = n % plan.b_stages;
                if (n >= 2) ok = tc::mbar_wait(&acc_empty[buf], (n / 2 - 1) & 1, s_abort, &g_lora_status, kWaitAccFree);
                if (ok) ok = tc::mbar_wait(&b_full[s], (n / plan.b_stages) & 1, s_abort, &g_lora_status, kWaitFull);
                if (!ok) break;
                tc::fence_after();
                for (int part = 0; part < 2; ++part)
                    for (int k = 0; k < k_steps; ++k)
                        tc::mma_16bit(tmem + buf * kN, tc::desc_lo(s_low + (part * plan.blocks + (k >> 2)) * kTileBytes) + 2 * (k & 3),
                                      tc::desc_lo(s_b + s * b_bytes + (k >> 2) * kN * 128) + 2 * (k & 3), id, part > 0 || k > 0);
                tc::commit(&b_empty[s]);
                tc::commit(&acc_full[buf]);
            }
        }
        if (!ok) {   // MMAs in flight end before the operands and the TMEM go
            tc::commit(drain);
            for (uint32_t i = 0; i < tc::kSpinLimit && !tc::mbar_try_wait(drain, 0); ++i) {}
        }
    } else {
        const int quarter = warp & 3, r_in_tile = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        uint32_t n = 0, yi = 0;
        bool ok = true;
        for (int64_t item = first; item < last && ok;) {
            const int64_t tile = item / plan.steps, begin = item - tile * plan.steps, end = min(plan.steps, begin + last - item);
            item += end - begin;
            int mine;
            const int count = tile_adapters(p, tile * kTile, lane, quarter, mine, nullptr);
            if (count == 0 && in_place) continue;
            const int64_t row = tile * kTile + r_in_tile;
            float factor = 0.0f;
            if (count > 0) {
                // (the tile before has been waited for accumulator by accumulator, so its MMAs are done with s_low)
                factor = put_low<T>(p, plan, s_low, row, r_in_tile, mine >= 0);
                if (mine >= 0 && p.scales) factor *= __ldg(p.scales + adapter_of(p, row));
                tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(low_full);
            }
            for (int64_t step = begin; step < end && ok; ++step, ++yi) {
                const int ys = yi % plan.y_stages;
                uint8_t* mine_y = s_y + ys * kYBytes + r_in_tile * 128;
                ok = tc::mbar_wait(&y_full[ys], (yi / plan.y_stages) & 1, s_abort, &g_lora_status, kWaitY);
                for (int j = 0; j < count && ok; ++j, ++n) {
                    const uint32_t buf = n & 1;
                    ok = tc::mbar_wait(&acc_full[buf], (n / 2) & 1, s_abort, &g_lora_status, kWaitAcc);
                    if (!ok) break;
                    tc::fence_after();
                    if (__any_sync(0xffffffffu, mine == j)) {
#pragma unroll
                        for (int c = 0; c < kN; c += 16) {
                            uint32_t v[16];
                            tc::ld16(tmem + lanes + buf * kN + c, v);
                            tc::wait_ld();
                            if (mine == j) {
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    uint4* at = reinterpret_cast<uint4*>(mine_y + (c >> 6) * kTileBytes + (((((c & 63) >> 3) + u) ^ (r_in_tile & 7)) << 4));
                                    Raw8<T> raw;
                                    raw.u = *at;
                                    float f[8];
                                    unpack8(raw, f);
#pragma unroll
                                    for (int i = 0; i < 8; ++i) f[i] = fmaf(factor, __uint_as_float(v[8 * u + i]), f[i]);
                                    *at = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
                                }
                            }
                        }
                    }
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
                }
                if (!ok) break;
                tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) {
#pragma unroll
                    for (int h = 0; h < kHalves; ++h)
                        tc::tma_store_2d(&map_out, s_y + ys * kYBytes + h * kTileBytes + quarter * 32 * 128, (int)(step * kN + h * 64),
                                         (int)(tile * kTile) + quarter * 32);
                    tc::tma_store_commit();
                    // a stage is handed back when its store has read it: one step later where there are stages to spare
                    if (plan.y_stages > 2) {
                        tc::tma_store_wait_read<1>();
                        if (yi > 0) tc::mbar_arrive(&y_empty[(yi - 1) % plan.y_stages]);
                    } else {
                        tc::tma_store_wait_read<0>();
                        tc::mbar_arrive(&y_empty[ys]);
                    }
                }
                __syncwarp();
            }
        }
        if (lane == 0) tc::tma_store_wait_read<0>();
        __syncwarp();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, 2 * kN);
}

// ------------------------------------------------------------------ host

int sm_count() {
    static int cached[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 148;
    if (cached[dev] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        cached[dev] = n > 0 ? n : 148;
    }
    return cached[dev];
}

bool few_rows(int64_t rows) { return rows <= 16; }

ShrinkPlan shrink_plan(int64_t rows, int64_t K, int64_t R, int64_t L) {
    ShrinkPlan s{};
    const int64_t tiles = ceil_div(rows, kTile), slots = 2 * sm_count();   // two CTAs an SM
    s.k_tiles = (int)ceil_div(K, 64);
    s.rn = (int)round_up(R, 16);
    int64_t splits = slots / tiles, most = s.k_tiles / 4;     // at least four steps of K each
    splits = splits > most ? most : splits;
    s.splits = (int)(splits < 1 ? 1 : splits > 65535 ? 65535 : splits);
    int64_t groups = slots / (tiles * s.splits), asked = rows < kTile ? rows : kTile;
    if (groups > asked) groups = asked;
    if (groups > L) groups = L;
    s.groups = (int)(groups < 1 ? 1 : groups);
    const int stage = kTileBytes + s.rn * 128;
    s.stages = (110 * 1024) / stage;
    if (s.stages > 6) s.stages = 6;
    s.accs = s.rn <= 128 ? 2 : 1;
    s.smem = 1024 + s.stages * (stage + 16) + 5 * 8 + kTile * 4 + 16;
    return s;
}

template <typename K>
int opt_in(K kernel, int which) {   // dynamic shared memory beyond 48 KB, once per kernel and device
    static bool done[8][64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[which][dev]) return CK_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e != cudaSuccess) CK_FAIL((int)e, "lora_add: cannot reserve %d bytes of shared memory: %s", kSmemMost, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[which][dev] = true;
    return CK_OK;
}

template <typename T, int kN>
int launch_expand(const LoraArgs& p, cudaStream_t stream) {
    ExpandPlan e{};
    e.steps = ceil_div(p.N, kN);
    e.items = e.steps * ceil_div(p.rows, kTile);
    e.blocks = (int)ceil_div(p.R, 64);
    const int b_bytes = e.blocks * kN * 128, y_bytes = kTile * kN * 2, rest = 1024 + 24 * 8 + kTile * 4 + 16;
    int room = kSmemMost - rest - 2 * e.blocks * kTileBytes;
    e.b_stages = e.y_stages = 2;
    room -= 2 * (b_bytes + y_bytes);
    for (int i = 0; i < 2; ++i) {
        if (room >= y_bytes) { ++e.y_stages; room -= y_bytes; }
        if (room >= b_bytes) { ++e.b_stages; room -= b_bytes; }
    }
    e.smem = kSmemMost - room;
    CUtensorMap map_b, map_y, map_out;
    const int64_t bd[3] = {p.R, p.N, p.L}, bs[2] = {p.R * 2, p.N * p.R * 2};
    const int64_t yd[2] = {p.N, p.rows}, ys[1] = {p.y_stride * 2}, os[1] = {p.out_stride * 2};
    if (!tc::make_map_16bit(&map_b, p.b, 3, bd, bs, kN) || !tc::make_map_16bit(&map_y, p.y, 2, yd, ys, kTile) ||
        !tc::make_map_16bit(&map_out, p.out, 2, yd, os, 32))
        CK_FAIL(CK_ERR_UNSUPPORTED, "lora_add: a tensor map could not be encoded");
    auto kernel = lora_expand_kernel<T, kN>;
    const int rc = opt_in(kernel, 1 + (Elem<T>::code == CK_BF16 ? 0 : 2) + (kN == 64));
    if (rc != CK_OK) return rc;
    const int64_t grid = e.items < sm_count() ? e.items : sm_count();
    kernel<<<(unsigned)grid, kThreads, e.smem, stream>>>(map_b, map_y, map_out, p, e);
    return launch_status("lora_add (expand)");
}

template <typename T>
int launch_many(LoraArgs p, cudaStream_t stream) {
    const ShrinkPlan s = shrink_plan(p.rows, p.K, p.R, p.L);
    p.splits = s.splits;
    CUtensorMap map_x, map_a;
    const int64_t xd[2] = {p.K, p.rows}, xs[1] = {p.x_stride * 2};
    const int64_t ad[3] = {p.K, p.R, p.L}, as[2] = {p.K * 2, p.R * p.K * 2};
    if (!tc::make_map_16bit(&map_x, p.x, 2, xd, xs, kTile) || !tc::make_map_16bit(&map_a, p.a, 3, ad, as, s.rn))
        CK_FAIL(CK_ERR_UNSUPPORTED, "lora_add: a tensor map could not be encoded");
    int rc = opt_in(lora_shrink_kernel, 0);
    if (rc != CK_OK) return rc;
    const dim3 grid((unsigned)ceil_div(p.rows, kTile), (unsigned)s.splits, (unsigned)s.groups);
    lora_shrink_kernel<<<grid, kThreads, s.smem, stream>>>(map_x, map_a, p, s, Elem<T>::code == CK_BF16);
    rc = launch_status("lora_add (shrink)");
    if (rc != CK_OK) return rc;
    return p.R <= 64 ? launch_expand<T, 128>(p, stream) : launch_expand<T, 64>(p, stream);
}

}  // namespace
}  // namespace ck

extern "C" int64_t ck_lora_workspace_bytes(int64_t rows, int64_t K, int64_t rank, int64_t adapters) {
    using namespace ck;
    if (rows <= 0 || K <= 0 || rank <= 0 || adapters <= 0 || few_rows(rows)) return 0;
    return shrink_plan(rows, K, rank, adapters).splits * rows * rank * 4;
}

extern "C" int ck_lora_device_status(void) {
    using namespace ck;
    int status = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&status, g_lora_status, sizeof(status));   // (synchronises)
    if (e != cudaSuccess) CK_FAIL((int)e, "ck_lora_device_status: %s", cudaGetErrorString(e));
    if (status == 0) return CK_OK;
    const int zero = 0;
    cudaMemcpyToSymbol(g_lora_status, &zero, sizeof(zero));
    CK_FAIL(CK_ERR_DEVICE_TIMEOUT, "lora_add: a bounded wait ran out (wait %d, CTA %d)", status >> 16, status & 0xffff);
}

extern "C" int launch_lora_add_kernel(const void* y, const void* x, const void* a, const void* b, const void* ids,
                                      const float* scales, void* out, void* workspace, int64_t rows, int64_t K, int64_t N,
                                      int64_t rank, int64_t adapters, int64_t y_row_stride, int64_t x_row_stride,
                                      int64_t out_row_stride, int64_t rows_per_id, int dtype_code, bool ids_64bit,
                                      cudaStream_t stream) {
    using namespace ck;
    if (!y || !x || !a || !b || !ids || !out) CK_FAIL(CK_ERR_NULL, "lora_add: null pointer");
    if (dtype_code != CK_F16 && dtype_code != CK_BF16) CK_FAIL(CK_ERR_DTYPE, "lora_add: dtype code %d (bf16 or fp16)", dtype_code);
    // (tiles are addressed with 32-bit coordinates; 2^27 rows keep the grid of the first product within its bounds)
    if (rows <= 0 || rows > (1 << 27) || K <= 0 || K > (1 << 30) || N <= 0 || N > (1 << 30) || adapters <= 0 || adapters > 0x7fffffff ||
        K % 8 != 0 || N % 8 != 0 || rows_per_id <= 0 || x_row_stride < K || y_row_stride < N || out_row_stride < N)
        CK_FAIL(CK_ERR_SHAPE, "lora_add: bad shape rows=%lld K=%lld N=%lld adapters=%lld (K and N multiples of 8)", (long long)rows,
                (long long)K, (long long)N, (long long)adapters);
    if (rank <= 0 || rank % 8 != 0 || rank > kMaxRank) CK_FAIL(CK_ERR_SHAPE, "lora_add: rank %lld (a multiple of 8, at most %d)", (long long)rank, kMaxRank);
    if (!aligned16(y) || !aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(out) || ((x_row_stride | y_row_stride | out_row_stride) & 7))
        CK_FAIL(CK_ERR_ALIGN, "lora_add: tensors and row strides must be 16-byte aligned");
    const LoraArgs p{y, x, a, b, ids, scales, out, static_cast<float*>(workspace), rows, K, N, rank, adapters, y_row_stride, x_row_stride, out_row_stride, rows_per_id, ids_64bit, 0};
    if (few_rows(rows)) {
        if (dtype_code == CK_BF16) lora_row_kernel<__nv_bfloat16><<<(unsigned)rows, 256, 0, stream>>>(p);
        else lora_row_kernel<__half><<<(unsigned)rows, 256, 0, stream>>>(p);
        return launch_status("lora_add");
    }
    if (!workspace) CK_FAIL(CK_ERR_NULL, "lora_add: a workspace of ck_lora_workspace_bytes() is needed");
    if (!aligned16(workspace)) CK_FAIL(CK_ERR_ALIGN, "lora_add: the workspace must be 16-byte aligned");
    return dtype_code == CK_BF16 ? launch_many<__nv_bfloat16>(p, stream) : launch_many<__half>(p, stream);
}
