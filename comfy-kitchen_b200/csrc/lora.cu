// Low-rank adapters of many requests beside a shared projection (sm_100a).
//
//   out[t] = y[t] + scale[a] * B_a (A_a x[t]),   a = ids[t];  out[t] = y[t] where a is no adapter (outside [0, L))
//
// y [T, N] is the shared projection's output for the rows x [T, K]; A_a [R, K], B_a [N, R].
//
// Bound by HBM in either direction: x is read once, y read and out written once (2 K + 4 N bytes a row), each used adapter
// once; the products' 2 R (K + N) flop a row stay below that up to a rank of about 128.  Two forms:
//   few rows:   a cluster of eight CTAs per row, one launch.
//   many rows:  four kernels, two of them on the tensor cores (tcgen05):
//               count:   which adapters each tile of rows asks for; by their number the others share out their work;
//               shrink:  low[t, :] = A x[t], equal shares of the tiles' K steps for every SM, partial sums in fp32;
//               join:    the partial sums added in order (no atomics, the same bits every time) and laid out as the
//                        next product's operand;
//               expand:  out = y + scale * (B low), y tiles fetched and out tiles stored by TMA while the products run.
// Ids are looked at on the device: a tile lists the adapters that its rows ask for, computes each one's product for all 128
// rows and keeps a row's own (a row of another request never enters a sum, whatever it holds).  Requests that lie behind
// one another cost nothing extra; a tile of 128 different adapters reads 128 adapters, as it must.
//
// Measured, back to back: 16384 rows, 8192 -> 8192, rank 128, 8 requests: 204 us (64 % of the copy rate; 186 in a short burst:
// the first product at 8, x done at 71, the sums joined at 81, the first output at 87); 4608 rows, 4096 -> 12288, rank 64, 7 requests: 76 us (54 %), of which
// about 30 are the four kernels' beginnings and ends; one row 4.0 us, 64 rows of 16 adapters 16.9 us on the device.
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
constexpr int kTileBytes = kTile * 128;   // 128 rows x 64 elements
constexpr int kSmemMost = 232448;

__device__ int g_lora_status = 0;
enum : int { kWaitFull = 1, kWaitEmpty = 2, kWaitAcc = 3, kWaitAccFree = 4, kWaitLow = 5, kWaitY = 6, kWaitYFree = 7, kWaitList = 8, kWaitDone = 9 };

constexpr int kShrinkRows = 256;    // rows of x in a tile of the first product (its MMA's N)

// What the rows of such a tile ask for.
struct alignas(16) TileList {
    int16_t slot[kShrinkRows];      // [token]: which adapter (-1: none)
    int id[kShrinkRows];            // [adapter]: its id,
    int16_t from[kShrinkRows];      // the first token (a multiple of 8)
    int16_t wide[kShrinkRows];      // and the number of tokens (of 16) that its product is taken for
    int count;
};

struct LoraArgs {
    const void* y;
    const void* x;
    const void* a;          // [L, R, K]
    const void* b;          // [L, N, R]
    const void* ids;        // int32 or int64, one per rows_per_id rows
    const float* scales;    // [L] or null
    void* out;
    uint8_t* image;         // many rows: per tile the low-rank vectors as the second product's operand (hi blocks, lo blocks)
    float* factor;          // [rows]: what a row's second product is multiplied by
    float* partial;         // [blocks, 256, R]: sums over a part of K for a tile of 256 rows
    int* asked128;          // [tiles of 128 rows]: how many adapters a tile asks for
    int* asked256;          // [tiles of 256 rows]
    int* list128;           // [tiles of 128 rows][128]: their ids
    int16_t* slot128;       // [tiles of 128 rows][128]: which of them a row asks for (-1: none)
    TileList* list256;      // [tiles of 256 rows]
    int* first_block;       // [tiles of 256 rows]: a tile's blocks in `partial`, first
    int* last_block;        // and last
    int64_t rows, K, N, R, L;
    int64_t y_stride, x_stride, out_stride;
    int64_t rows_per_id;
    int ids64;
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

constexpr int kFewCluster = 8, kFewThreads = 256, kFewWarps = kFewThreads / 32;

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// A cluster of eight CTAs per row, one launch: each CTA sums its eighth of K for the whole low-rank vector, hands that to
// the others through their shared memory, and computes its eighth of the output's columns.  What it costs is latency
// (ids, A, the exchange, B), so B and y are fetched into L2 meanwhile.  Rows of one adapter read it from L2 again.
template <typename T>
__global__ void __cluster_dims__(kFewCluster, 1, 1) __launch_bounds__(kFewThreads)
lora_few_kernel(const LoraArgs p) {
    __shared__ __align__(16) float s_part[kFewWarps][kMaxRank];      // [part of this CTA's K][r]
    __shared__ __align__(16) float s_all[kFewCluster][kMaxRank];     // [CTA][r], written by all of them
    __shared__ __align__(16) float s_low[kMaxRank];
    const int64_t row = blockIdx.y;
    const int rank = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, R = (int)p.R;
    const T* y = static_cast<const T*>(p.y) + row * p.y_stride;
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    const int n0 = (int)(p.N / 8 * rank / kFewCluster) * 8, n1 = (int)(p.N / 8 * (rank + 1) / kFewCluster) * 8;
    const int id = adapter_of(p, row);
    if (id < 0) {   // (the same for the whole cluster)
        if (p.out != p.y)
            for (int n = n0 + tid * 8; n < n1; n += kFewThreads * 8) *reinterpret_cast<uint4*>(out + n) = *reinterpret_cast<const uint4*>(y + n);
        return;
    }
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (waited for before the first store to another CTA)
    const T* b = static_cast<const T*>(p.b) + ((int64_t)id * p.N + n0) * R;
    for (int i = tid; i < ((n1 - n0) * R + 63) / 64; i += kFewThreads) prefetch_l2(b + (int64_t)i * 64);
    for (int i = tid; i < (n1 - n0 + 63) / 64; i += kFewThreads) prefetch_l2(y + n0 + i * 64);
    const float scale = p.scales ? __ldg(p.scales + id) : 1.0f;

    // four rows of A a warp at a time; where that leaves warps over, they share the K part
    const int fours = R / 4;
    const int parts = fours >= kFewWarps ? 1 : kFewWarps / fours;
    const int part = warp / (kFewWarps / parts), member = warp % (kFewWarps / parts), members = kFewWarps / parts;
    const int c0 = (int)(p.K / 8 * (rank * parts + part) / (kFewCluster * parts)), c1 = (int)(p.K / 8 * (rank * parts + part + 1) / (kFewCluster * parts));
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* a = static_cast<const T*>(p.a) + (int64_t)id * R * p.K;
    for (int four = member; four < fours; four += members) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const T* ar = a + (int64_t)four * 4 * p.K;
#pragma unroll 2
        for (int c = c0 + lane; c < c1; c += 32) {
            float u[8], v[4][8];
            load8<T>(x + c * 8, u);
#pragma unroll
            for (int i = 0; i < 4; ++i) load8<T>(ar + i * p.K + c * 8, v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[i] = fmaf(u[j], v[i][j], sum[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = warp_sum(sum[i]);
        if (lane == 0) *reinterpret_cast<float4*>(&s_part[part][four * 4]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int i = tid; i < R * kFewCluster; i += kFewThreads) {
        const int to = i / R, r = i - to * R;
        float v = s_part[0][r];
        for (int k = 1; k < parts; ++k) v += s_part[k][r];
        uint32_t addr;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(tc::smem_u32(&s_all[rank][r])), "r"(to));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
    }
    tc::cluster_sync();
    for (int r = tid; r < R; r += kFewThreads) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kFewCluster; ++k) v += s_all[k][r];
        s_low[r] = v;
    }
    __syncthreads();
#pragma unroll 2
    for (int n = tid; n < n1 - n0; n += kFewThreads) {
        const float base = Elem<T>::to_f32(y[n0 + n]);
        float sum = 0.0f;
        for (int r = 0; r < R; r += 8) {
            float v[8];
            load8<T>(b + (int64_t)n * R + r, v);
            const float4 lo = *reinterpret_cast<const float4*>(s_low + r), hi = *reinterpret_cast<const float4*>(s_low + r + 4);
            sum = fmaf(lo.x, v[0], sum); sum = fmaf(lo.y, v[1], sum); sum = fmaf(lo.z, v[2], sum); sum = fmaf(lo.w, v[3], sum);
            sum = fmaf(hi.x, v[4], sum); sum = fmaf(hi.y, v[5], sum); sum = fmaf(hi.z, v[6], sum); sum = fmaf(hi.w, v[7], sum);
        }
        out[n0 + n] = Elem<T>::from_f32(fmaf(scale, sum, base));
    }
}

// ------------------------------------------------------------------ many rows

// The ids that kRows rows from row0 on ask for (-1: none): lane l has rows l, l + 32, ...
template <int kRows>
__device__ __forceinline__ void tile_ids(const LoraArgs& p, int64_t row0, int lane, int (&id)[kRows / 32]) {
#pragma unroll
    for (int q = 0; q < kRows / 32; ++q) {
        const int64_t row = row0 + 32 * q + lane;
        id[q] = row < p.rows ? adapter_of(p, row) : -1;
    }
}

// The different adapters among them, in the order of their first rows: calls each(place, id, first row, last row) with
// every lane, leaves each row's place in `slot` (-1: none) and returns their number.  By a whole warp.
template <int kRows, typename Each>
__device__ __forceinline__ int tile_adapters(const int (&id)[kRows / 32], int lane, int16_t* slot, Each each) {
    constexpr int kQ = kRows / 32;
    int place[kQ];
    uint32_t left[kQ], any = 0;
#pragma unroll
    for (int q = 0; q < kQ; ++q) { any |= left[q] = __ballot_sync(0xffffffffu, id[q] >= 0); place[q] = -1; }
    int count = 0;
    while (any) {
        int cur = -1, lo = 0, hi = 0;
#pragma unroll
        for (int q = kQ - 1; q >= 0; --q) {   // (the first 32 rows that have one left decide)
            const int first = __shfl_sync(0xffffffffu, id[q], left[q] ? __ffs(left[q]) - 1 : 0);
            if (left[q]) { cur = first; lo = 32 * q + __ffs(left[q]) - 1; }
        }
        any = 0;
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            const uint32_t same = __ballot_sync(0xffffffffu, id[q] == cur);
            if (same) hi = 32 * q + 31 - __clz(same);
            if (id[q] == cur) place[q] = count;
            any |= left[q] &= ~same;
        }
        each(count, cur, lo, hi);
        ++count;
    }
#pragma unroll
    for (int q = 0; q < kQ; ++q)
        slot[32 * q + lane] = (int16_t)place[q];
    return count;
}

// ---- shares: tiles ask for different numbers of adapters and cost accordingly, so a CTA's share is an equal run of weighted
// steps, a tile's being `steps` steps of the weight that its number of adapters has (nought: the tile needs no work).

struct Place { int tile, step, worked; };   // `worked`: how many tiles before have work

// Where position `pos` of all tiles' weighted steps lies.  By a whole warp.
template <typename Weight>
__device__ __forceinline__ Place locate(const int* asked, int tiles, int steps, int64_t pos, int lane, Weight weight) {
    int64_t before = 0;
    int worked = 0;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const int w = t0 + lane < tiles ? weight(__ldcg(asked + t0 + lane)) : 0;
        int upto = w;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, w > 0 && pos < (before + upto) * steps);
        const uint32_t work = __ballot_sync(0xffffffffu, w > 0);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const int wt = __shfl_sync(0xffffffffu, w, l);
            const int64_t start = (before + __shfl_sync(0xffffffffu, upto, l) - wt) * steps;
            return Place{t0 + l, (int)((pos - start) / wt), worked + __popc(work & ((1u << l) - 1))};
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        worked += __popc(work);
    }
    return Place{tiles, 0, worked};   // (the end)
}

// All tiles' weight, and how many of them have work.  By a whole warp.
template <typename Weight>
__device__ __forceinline__ int64_t total_weight(const int* asked, int tiles, int lane, int& worked, Weight weight) {
    int64_t sum = 0;
    worked = 0;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const int w = t0 + lane < tiles ? weight(__ldcg(asked + t0 + lane)) : 0;
        worked += __popc(__ballot_sync(0xffffffffu, w > 0));
        sum += w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// One CTA per 256 rows: warps 0 and 1 list a half's adapters, warp 2 the whole tile's.  (The kernels behind read the lists; working
// them out again there, with code that no cache holds yet, took 4 us before the first product.)
__global__ void __launch_bounds__(96) lora_count_kernel(const LoraArgs p) {
    tc::launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tile = blockIdx.x;
    if (warp < 2) {
        const int64_t half = tile * 2 + warp;
        int id[4];
        tile_ids<kTile>(p, half * kTile, lane, id);
        const int n = tile_adapters<kTile>(id, lane, p.slot128 + half * kTile, [&](int j, int which, int, int) { if (lane == 0) p.list128[half * kTile + j] = which; });
        if (lane == 0) p.asked128[half] = n;
    } else {
        TileList& l = p.list256[tile];
        int id[8];
        tile_ids<kShrinkRows>(p, tile * kShrinkRows, lane, id);
        const int n = tile_adapters<kShrinkRows>(id, lane, l.slot, [&](int j, int which, int lo, int hi) {
            const int wide = (hi + 1 - (lo & ~7) + 15) & ~15;
            if (lane == 0) { l.id[j] = which; l.wide[j] = (int16_t)wide; l.from[j] = (int16_t)min(lo & ~7, kShrinkRows - wide); }
        });
        // (no blocks, until the first product's kernel says otherwise: one that gives up may not)
        if (lane == 0) { l.count = n; p.asked256[tile] = n; p.first_block[tile] = 0; p.last_block[tile] = -1; }
    }
}

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

// fp16: the power of two that brings a row of largest magnitude `most` to [1, 2), and its inverse.
__device__ __forceinline__ void row_scale(float most, float& down, float& up) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127;   // most is in [2^e, 2^(e+1))
    down = up = 1.0f;
    if (e < 127 && e > -126) {                                // (not for zeros, infinities and what fp32 itself barely holds)
        up = __uint_as_float((uint32_t)(e + 127) << 23);
        down = __uint_as_float((uint32_t)(127 - e) << 23);
    }
}

// Elements r .. r + 7 of row `row` of a tile's image: hi and lo parts, in the swizzled order in which the MMA reads shared
// memory, so that the second kernel fetches a tile with one bulk copy.
template <typename T>
__device__ __forceinline__ void put_image(uint8_t* image, int blocks, int row, int r, const float (&v)[8], float down) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = v[2 * i] * down, b = v[2 * i + 1] * down;
        const float ha = Elem<T>::round(a), hb = Elem<T>::round(b);
        hi[i] = pack2<T>(ha, hb);
        lo[i] = pack2<T>(isfinite(ha) ? a - ha : 0.0f, isfinite(hb) ? b - hb : 0.0f);   // (an infinity stays one)
    }
    uint8_t* dst = image + (r >> 6) * kTileBytes + row * 128 + ((((r & 63) >> 3) ^ (row & 7)) << 4);
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(dst + blocks * kTileBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

struct ShrinkPlan {
    int k_tiles, halves;        // 64-element steps of K; 128-row tiles of A (2 for ranks over 128)
    int blocks;                 // 64-element blocks of R
    int tiles, ctas;            // tiles of 256 rows; CTAs
    int x_stages, a_stages;     // rings of x and A tiles
    int smem;
};

constexpr int kShrinkThreads = 352;        // warp 0: TMA, warp 1: MMA, warps 2-9: epilogue, warp 10: the tiles' lists
constexpr int kXBytes = kShrinkRows * 128;
constexpr int kShrinkColumns = 512;        // all of TMEM

// A K step of a tile of two adapters takes about 5/4 of the time of one of a single adapter's, of three 7/4 (fewer steps of x
// fit ahead of the A tiles' ring), and so on.  (The weight ends at 16, four times the least one: with at least four steps a CTA on
// average, no share is then shorter than a step.)
__device__ __forceinline__ int shrink_weight(int asked) { return asked == 0 ? 0 : asked < 3 ? 3 + asked : min(2 * asked + 1, 16); }

// low[t][:] = A_{ids[t]} x[t] as partial sums over parts of K: every CTA takes an equal run of the tiles' K steps, so that all
// SMs are busy whatever the number of rows, and leaves a block of sums for each tile that it meets.  CTA c's block for
// the n-th tile that has work is block c + n: of two neighbouring blocks either the CTA or the tile is another one.
//
// The product is taken as A x^T: an MMA of 128 rows costs 128 clocks whether it has 64 columns or 256, so the rank is its M
// (what lies behind it in shared memory only fills accumulator rows that nobody reads) and 256 tokens its N; with the roles
// the other way round the tensor cores, not memory, were the bound.  The accumulator holds a token per column, and its 32
// lanes store consecutive elements of a token's vector.
// Adapters share a pass over x as long as their accumulators fit TMEM.  An adapter's product is taken only for the tokens
// from the first to the last that asks for it, so requests that lie behind one another fit by the dozen: a tile in which
// some meet costs their A tiles (from L2), not a second read of x.
template <typename T>
__global__ void __launch_bounds__(kShrinkThreads, 1)
lora_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const LoraArgs p,
                   const ShrinkPlan plan) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int a_bytes = plan.halves * kTileBytes;
    const uint32_t a_tx = (uint32_t)p.R * 128;                                // (rows of A behind the rank are not fetched)
    uint8_t* s_x = smem;
    uint8_t* s_a = s_x + plan.x_stages * kXBytes;
    uint64_t* x_full = reinterpret_cast<uint64_t*>(s_a + plan.a_stages * a_bytes);
    uint64_t* x_empty = x_full + plan.x_stages;
    uint64_t* a_full = x_empty + plan.x_stages;
    uint64_t* a_empty = a_full + plan.a_stages;
    uint64_t* acc_full = a_empty + plan.a_stages;
    uint64_t* acc_empty = acc_full + 1;
    uint64_t* drain = acc_empty + 1;
    uint64_t* listed = drain + 1;                                             // [2] a tile's lists are there
    uint64_t* unlisted = listed + 2;                                          // [2] nobody needs them any more
    TileList* s_lists = reinterpret_cast<TileList*>((reinterpret_cast<uintptr_t>(unlisted + 2) + 15) & ~uintptr_t(15));   // [2]
    Place* s_share = reinterpret_cast<Place*>(s_lists + 2);                   // this CTA's: from, to
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_share + 2);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 1) {
        tc::tmem_alloc(s_tmem, kShrinkColumns);
    } else if (threadIdx.x == 0) {
        for (int s = 0; s < plan.x_stages; ++s) { tc::mbar_init(&x_full[s], 1); tc::mbar_init(&x_empty[s], 1); }
        for (int s = 0; s < plan.a_stages; ++s) { tc::mbar_init(&a_full[s], 1); tc::mbar_init(&a_empty[s], 1); }
        tc::mbar_init(acc_full, 1);
        tc::mbar_init(acc_empty, 8);
        tc::mbar_init(drain, 1);
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&listed[i], 1); tc::mbar_init(&unlisted[i], 10); }
        *s_abort = 0;
        tc::mbar_init_done();
    } else if (warp == 2) {
        tc::wait_for_dependency();      // the counts
        int worked;
        const int64_t all = total_weight(p.asked256, plan.tiles, lane, worked, shrink_weight) * plan.k_tiles;
        const int sharing = min(plan.ctas, max(1, worked * plan.k_tiles / 4));   // (at least four steps a CTA)
        const int cta = min((int)blockIdx.x, sharing);
        const Place from = locate(p.asked256, plan.tiles, plan.k_tiles, all * cta / sharing, lane, shrink_weight);
        const Place to = locate(p.asked256, plan.tiles, plan.k_tiles, all * min(cta + 1, sharing) / sharing, lane, shrink_weight);
        if (lane == 0) { s_share[0] = from; s_share[1] = to; }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    tc::launch_dependents();
    const uint32_t tmem = *s_tmem;
    const Place from = s_share[0], to = s_share[1];
    const bool idle = from.tile == to.tile && from.step == to.step;
    const int tile0 = from.tile, tile1 = idle ? tile0 - 1 : to.step > 0 ? to.tile : to.tile - 1;   // (the last one that has steps of this share)

    if (warp == 10) {
        // lists, a tile ahead of the other warps
        bool ok = true;
        for (int tile = tile0; tile <= tile1 && ok; ++tile) {
            const int at = (tile - tile0) & 1;
            TileList& l = s_lists[at];
            const TileList& from_count = p.list256[tile];
            // (a lane's share of the slots, of the first 32 adapters and the count at once)
            const uint4 slots = __ldcg(reinterpret_cast<const uint4*>(from_count.slot) + lane);
            const int found = __ldcg(&from_count.count);
            int id = __ldcg(from_count.id + lane);
            int16_t first = __ldcg(from_count.from + lane), wide = __ldcg(from_count.wide + lane);
            ok = tc::mbar_wait(&unlisted[at], ((tile - tile0) >> 1 & 1) ^ 1, s_abort, &g_lora_status, kWaitList);
            if (!ok) break;
            reinterpret_cast<uint4*>(l.slot)[lane] = slots;
            for (int j = lane;;) {
                l.id[j] = id;
                l.from[j] = first;
                l.wide[j] = wide;
                if ((j += 32) >= found) break;
                id = __ldcg(from_count.id + j);
                first = __ldcg(from_count.from + j);
                wide = __ldcg(from_count.wide + j);
            }
            if (lane == 0) l.count = found;
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&listed[at]);
            __syncwarp();
        }
    }
    tc::Ring xr, ar;
    uint32_t xs = 0, as = 0, n = 0;     // tiles issued (warp 0); accumulator rounds
    // x's first tiles are on their way before the ids are listed
    int ahead = 0;
    if (warp == 0) {
        const int k0 = from.step, k1 = tile0 == to.tile ? to.step : plan.k_tiles;
        for (; ahead < min(plan.x_stages, k1 - k0) && tile0 <= tile1; ++ahead) {
            if (tc::elect_one()) {
                tc::mbar_expect_tx(&x_full[ahead], kXBytes);
                tc::tma_load_2d(s_x + ahead * kXBytes, &map_x, (k0 + ahead) * 64, tile0 * kShrinkRows, &x_full[ahead]);
            }
            __syncwarp();
        }
    }
    bool ok = true;
    int block = (int)blockIdx.x + from.worked;
    for (int tile = tile0; tile <= tile1 && ok && warp < 10; ++tile) {
        const int at = (tile - tile0) & 1;
        const int k0 = tile == tile0 ? from.step : 0, k1 = tile == to.tile ? to.step : plan.k_tiles;
        ok = tc::mbar_wait(&listed[at], (tile - tile0) >> 1 & 1, s_abort, &g_lora_status, kWaitList);
        const TileList& l = s_lists[at];
        const int count = ok ? l.count : 0;
        // a batch: adapters `first` to `until`, their accumulators side by side
        auto batch_end = [&](int first) {
            int until = first, columns = 0;
            while (until < count && (columns += plan.halves * l.wide[until]) <= kShrinkColumns) ++until;
            return until;
        };
        if (warp == 0) {
            for (int first = 0, until; first < count && ok; first = until) {
                until = batch_end(first);
                for (int kt = k0; kt < k1 && ok; ++kt) {
                    if (ahead > 0) --ahead;
                    else {
                        ok = tc::mbar_wait(&x_empty[xr.at], xr.round ^ 1u, s_abort, &g_lora_status, kWaitEmpty);
                        if (!ok) break;
                        if (tc::elect_one()) {
                            tc::mbar_expect_tx(&x_full[xr.at], kXBytes);
                            tc::tma_load_2d(s_x + xr.at * kXBytes, &map_x, kt * 64, tile * kShrinkRows, &x_full[xr.at]);
                        }
                        __syncwarp();
                    }
                    ++xs;
                    xr.next(plan.x_stages);
                    for (int j = first; j < until; ++j) {
                        ok = tc::mbar_wait(&a_empty[ar.at], ar.round ^ 1u, s_abort, &g_lora_status, kWaitEmpty);
                        if (!ok) break;
                        const int which = l.id[j];
                        if (tc::elect_one()) {
                            tc::mbar_expect_tx(&a_full[ar.at], a_tx);
                            tc::tma_load_3d(s_a + ar.at * a_bytes, &map_a, kt * 64, 0, which, &a_full[ar.at]);
                        }
                        __syncwarp();
                        ++as;
                        ar.next(plan.a_stages);
                    }
                }
            }
        } else if (warp == 1) {
            for (int first = 0, until; first < count && ok; first = until, ++n) {
                until = batch_end(first);
                ok = tc::mbar_wait(acc_empty, (n & 1) ^ 1, s_abort, &g_lora_status, kWaitAccFree);
                for (int kt = k0; kt < k1 && ok; ++kt, xr.next(plan.x_stages)) {
                    ok = tc::mbar_wait(&x_full[xr.at], xr.round, s_abort, &g_lora_status, kWaitFull);
                    uint32_t d = tmem;
                    for (int j = first; j < until && ok; ++j, ar.next(plan.a_stages)) {
                        ok = tc::mbar_wait(&a_full[ar.at], ar.round, s_abort, &g_lora_status, kWaitFull);
                        if (!ok) break;
                        tc::fence_after();
                        const int wide = l.wide[j];
                        const uint32_t tokens = l.from[j], desc = tc::idesc(Elem<T>::code == CK_BF16, wide);
                        if (tc::elect_one()) {
                            const uint32_t da = tc::desc_lo(s_a + ar.at * a_bytes), db = tc::desc_lo(s_x + xr.at * kXBytes + tokens * 128);
                            for (int h = 0; h < plan.halves; ++h)
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    tc::mma_16bit(d + h * wide, da + h * (kTileBytes >> 4) + 2 * k, db + 2 * k, desc, kt > k0 || k > 0);
                            tc::commit(&a_empty[ar.at]);
                            if (j + 1 == until) {
                                tc::commit(&x_empty[xr.at]);
                                if (kt + 1 == k1) tc::commit(acc_full);
                            }
                        }
                        __syncwarp();
                        d += plan.halves * wide;
                    }
                }
            }
        } else {
            // a warp: 32 elements of the vector (its TMEM lanes) of every other 16 tokens
            const int quarter = warp & 3, half = (warp - 2) >> 2;
            float* part = p.partial + (int64_t)block * kShrinkRows * p.R;
            if (threadIdx.x == 64 && count > 0) {
                if (k0 == 0) p.first_block[tile] = block;
                if (k1 == plan.k_tiles) p.last_block[tile] = block;
            }
            const int R = (int)p.R;
            for (int first = 0, until; first < count && ok; first = until, ++n) {
                until = batch_end(first);
                ok = tc::mbar_wait(acc_full, n & 1, s_abort, &g_lora_status, kWaitAcc);
                if (!ok) break;
                tc::fence_after();
                uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
                for (int j = first; j < until; ++j) {
                    const int wide = l.wide[j], from = l.from[j];
                    for (int h = 0; h < plan.halves; ++h, acc += wide) {
                        const int r = h * kTile + quarter * 32 + lane;
                        if (r - lane >= R) continue;
                        float* dst = part + (from + half * 16) * R + r;
                        for (int t = half * 16; t < wide; t += 32, dst += 32 * R) {
                            const uint32_t asked = __ballot_sync(0xffffffffu, lane < 16 && l.slot[from + t + (lane & 15)] == j);
                            if (!asked) continue;
                            uint32_t v[16];
                            tc::ld16(acc + t, v);
                            tc::wait_ld();
                            float* to = dst;
                            if (asked == 0xffffu) {
                                if (r < R) {
#pragma unroll
                                    for (int i = 0; i < 16; ++i, to += R) *to = __uint_as_float(v[i]);
                                }
                            } else if (r < R) {
#pragma unroll
                                for (int i = 0; i < 16; ++i, to += R)
                                    if (asked >> i & 1) *to = __uint_as_float(v[i]);
                            }
                        }
                    }
                }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(acc_empty);
            }
        }
        block += count > 0;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&unlisted[at]);
    }
    if (!ok) {   // given up: copies and MMAs in flight end before shared memory and TMEM go
        if (warp == 0) {
            for (; ahead > 0; --ahead, ++xs) xr.next(plan.x_stages);
            tc::ring_drain(x_full, xr, xs, plan.x_stages);
            tc::ring_drain(a_full, ar, as, plan.a_stages);
        } else if (warp == 1) {
            if (tc::elect_one()) tc::commit(drain);
            __syncwarp();
            tc::mbar_drain(drain, 0);
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, kShrinkColumns);
}

// The parts of K, added up in their order and written as the image that the second product reads: eight lanes a token, each
// with every eighth chunk of 8 elements.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) lora_join_kernel(const LoraArgs p, const ShrinkPlan plan) {
    tc::launch_dependents();
    const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / 8) + (threadIdx.x >> 3);
    const int sub = threadIdx.x & 7;
    // (the lists, as all others use them, not the ids: a tile that nobody asked anything of then has no sums)
    const int place = row < p.rows ? __ldcg(p.slot128 + row) : -1;
    const int id = place >= 0 ? __ldcg(p.list128 + row / kTile * kTile + place) : -1;
    const float scale = id >= 0 && p.scales ? __ldg(p.scales + id) : 1.0f;
    tc::wait_for_dependency();
    // (where the first product's kernel has given up on a tile, either may still be what the count kernel has set: no blocks, or some
    // of another tile's, but none outside `partial`; the status word says that the result is none)
    const int tile = (int)(row / kShrinkRows), block0 = id >= 0 ? __ldcg(p.first_block + tile) : 0, block1 = id >= 0 ? __ldcg(p.last_block + tile) : -1;
    float v[kMaxRank / 64][8];
#pragma unroll
    for (int u = 0; u < kMaxRank / 64; ++u) {
        const int c = (u * 8 + sub) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
        if (id >= 0 && c < p.R) {
            const float* src = p.partial + ((int64_t)block0 * kShrinkRows + row % kShrinkRows) * p.R + c;
#pragma unroll 4
            for (int k = block0; k <= block1; ++k, src += kShrinkRows * p.R) {
                const float4 a = __ldcg(reinterpret_cast<const float4*>(src)), b = __ldcg(reinterpret_cast<const float4*>(src) + 1);
                v[u][0] += a.x; v[u][1] += a.y; v[u][2] += a.z; v[u][3] += a.w;
                v[u][4] += b.x; v[u][5] += b.y; v[u][6] += b.z; v[u][7] += b.w;
            }
        }
    }
    float down = 1.0f, up = 1.0f;
    if (Elem<T>::code == CK_F16) {
        float most = 0.0f;
#pragma unroll
        for (int u = 0; u < kMaxRank / 64; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[u][i]));
#pragma unroll
        for (int o = 1; o < 8; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        row_scale(most, down, up);
    }
    if (id < 0) return;
    uint8_t* image = p.image + row / kTile * (2 * plan.blocks * kTileBytes);
    const int padded = (int)round_up(p.R, 16);   // (the second product's steps)
#pragma unroll
    for (int u = 0; u < kMaxRank / 64; ++u)
        if ((u * 8 + sub) * 8 < padded) put_image<T>(image, plan.blocks, (int)(row % kTile), (u * 8 + sub) * 8, v[u], down);
    if (sub == 0) p.factor[row] = scale * up;
}

struct ExpandPlan {
    int steps, tiles;           // column steps of a tile; tiles of 128 rows
    int k_steps;                // 16-element steps of R
    int blocks;                 // 64-element blocks of R
    int b_stages, y_stages;
    int smem;
};

constexpr int kEpiGroups = 2;              // units of 64 columns are dealt to two groups of four epilogue warps
constexpr int kExpandThreads = 128 + kEpiGroups * 128;  // warp 0: y's tiles, 1: MMA, 2-9: epilogue, 10: B's tiles, 11: stores

// Persistent CTAs take equal runs of (tile, column step) items; a step is kU units of 64 columns.  The MMA of 128 rows
// costs 128 clocks however few columns it has, and reads its 128 rows of the image from shared memory each time, so steps
// have two units unless that leaves SMs without an item (the whole call for 16384 x 8192, rank 128: 204 us, with one unit
// 235; 4608 x 12288, rank 64: 76 and 80).  Three or four units leave no room to fetch y ahead.  With the vectors in tensor
// memory instead, put there by the epilogue warps, there is room, but a tile begins later: 207 and 81 us.
template <typename T, int kU>
__global__ void __launch_bounds__(kExpandThreads, 1)
lora_expand_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_y,
                   const __grid_constant__ CUtensorMap map_out, const LoraArgs p, const ExpandPlan plan) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int kStep = kU * 64, kExpandColumns = 2 * kStep;
    constexpr int b_bytes = kStep * 128;                               // 64 elements of R for a step's columns
    const uint32_t low_bytes = 2 * plan.blocks * kTileBytes;
    uint8_t* s_low = smem;                                             // hi blocks, lo blocks
    uint8_t* s_b = s_low + low_bytes;
    uint8_t* s_y = s_b + plan.b_stages * b_bytes;
    uint64_t* b_full = reinterpret_cast<uint64_t*>(s_y + plan.y_stages * kTileBytes);
    uint64_t* b_empty = b_full + plan.b_stages;
    uint64_t* y_full = b_empty + plan.b_stages;
    uint64_t* y_empty = y_full + plan.y_stages;
    uint64_t* y_done = y_empty + plan.y_stages;                        // a unit's result is in its stage
    uint64_t* acc_full = y_done + plan.y_stages;                       // [2]
    uint64_t* acc_empty = acc_full + 2;                                // [2]
    uint64_t* low_full = acc_empty + 2;
    uint64_t* low_done = low_full + 1;                                 // a tile's last MMA is complete
    uint64_t* drain = low_done + 1;
    int* s_list = reinterpret_cast<int*>(drain + 1);                   // (warp 10's)
    Place* s_share = reinterpret_cast<Place*>(s_list + kTile);         // this CTA's: from, to
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_share + 2);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool in_place = p.out == p.y;

    if (threadIdx.x == 64) {
        for (int s = 0; s < plan.b_stages; ++s) { tc::mbar_init(&b_full[s], 1); tc::mbar_init(&b_empty[s], 1); }
        for (int s = 0; s < plan.y_stages; ++s) { tc::mbar_init(&y_full[s], 1); tc::mbar_init(&y_empty[s], 1); tc::mbar_init(&y_done[s], 4); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 4 * kEpiGroups); }
        tc::mbar_init(low_full, 1);
        tc::mbar_init(low_done, 1);
        tc::mbar_init(drain, 1);
        *s_abort = 0;
        tc::mbar_init_done();
    }
    if (warp == 1) tc::tmem_alloc(s_tmem, kExpandColumns);
    if (warp == 3) {
        // (The counts are there: this kernel can start only when every CTA of the two before it has, and the first of those
        // waits for them.)  In units of 128 clocks: an item's share of HBM's time, three quarters as much again for each further
        // adapter (ranks 64 and 128) and a third less without one, or the MMAs of a high rank.
        const int mmas = kU * plan.k_steps + 1;
        auto weight = [&](int asked) { return asked == 0 ? (in_place ? 0 : 7 * kU) : max(11 * kU * (3 * asked + 1) / 4, asked * mmas); };
        int worked;
        const int64_t all = total_weight(p.asked128, plan.tiles, lane, worked, weight) * plan.steps;
        const Place from = locate(p.asked128, plan.tiles, plan.steps, all * blockIdx.x / gridDim.x, lane, weight);
        const Place to = locate(p.asked128, plan.tiles, plan.steps, all * (blockIdx.x + 1) / gridDim.x, lane, weight);
        if (lane == 0) { s_share[0] = from; s_share[1] = to; }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *s_tmem;
    const Place from = s_share[0], to = s_share[1];
    const bool idle = from.tile == to.tile && from.step == to.step;
    const int tile1 = idle ? from.tile - 1 : to.step > 0 ? to.tile : to.tile - 1;   // the last tile that has steps of this share
    auto begin_of = [&](int tile) { return tile == from.tile ? from.step : 0; };
    auto end_of = [&](int tile) { return tile == to.tile ? to.step : plan.steps; };

    auto tile_count = [&](int tile) { return __ldcg(p.asked128 + tile); };
    // y's and B's tiles come from two warps: what frees a y tile needs products, and what frees a B tile may need y tiles.
    // A full ring is not freed before the kernels that this one hangs on are done, and those may run on for longer than a bounded
    // wait lasts (a CTA starts here as soon as its SM is free, and tiles that hundreds of adapters meet in keep others busy): so
    // every role waits for them first, without a limit, and counts only from there.
    if (warp == 0) {
        tc::Ring yr;
        uint32_t issued = 0;
        bool ok = true;
        for (int tile = from.tile; tile <= tile1 && ok; ++tile) {
            const int begin = begin_of(tile), end = end_of(tile);
            if (in_place && tile_count(tile) == 0) continue;
            for (int unit = begin * kU; unit < end * kU; ++unit) {
                if (issued == (uint32_t)plan.y_stages) tc::wait_for_dependency();   // (see above)
                ok = tc::mbar_wait(&y_empty[yr.at], yr.round ^ 1u, s_abort, &g_lora_status, kWaitYFree);
                if (!ok) break;
                if (tc::elect_one()) {
                    tc::mbar_expect_tx(&y_full[yr.at], kTileBytes);
                    tc::tma_load_2d(s_y + yr.at * kTileBytes, &map_y, unit * 64, tile * kTile, &y_full[yr.at]);
                }
                __syncwarp();
                ++issued;
                yr.next(plan.y_stages);
            }
        }
        if (!ok) tc::ring_drain(y_full, yr, issued, plan.y_stages);
    } else if (warp == 10) {
        tc::Ring br;
        uint32_t issued = 0;
        bool ok = true;
        for (int tile = from.tile; tile <= tile1 && ok; ++tile) {
            const int begin = begin_of(tile), end = end_of(tile);
            const int count = tile_count(tile);
            for (int j = lane; j < count; j += 32) s_list[j] = __ldcg(p.list128 + (int64_t)tile * kTile + j);
            __syncwarp();
            for (int step = begin; step < end && ok; ++step)
                for (int j = 0; j < count && ok; ++j) {
                    const int which = s_list[j];
                    for (int k = 0; k < plan.blocks; ++k) {
                        if (issued == (uint32_t)plan.b_stages) tc::wait_for_dependency();
                        ok = tc::mbar_wait(&b_empty[br.at], br.round ^ 1u, s_abort, &g_lora_status, kWaitEmpty);
                        if (!ok) break;
                        if (tc::elect_one()) {
                            tc::mbar_expect_tx(&b_full[br.at], (uint32_t)b_bytes);
                            tc::tma_load_3d(s_b + br.at * b_bytes, &map_b, k * 64, step * kStep, which, &b_full[br.at]);
                        }
                        __syncwarp();
                        ++issued;
                        br.next(plan.b_stages);
                    }
                }
        }
        if (!ok) tc::ring_drain(b_full, br, issued, plan.b_stages);
    } else if (warp == 1) {
        const uint32_t desc = tc::idesc(Elem<T>::code == CK_BF16, kStep);
        const int k_steps = plan.k_steps;
        tc::Ring br;
        uint32_t n = 0, seg = 0;
        bool ok = true;
        for (int tile = from.tile; tile <= tile1 && ok; ++tile) {
            const int begin = begin_of(tile), end = end_of(tile);
            const int count = tile_count(tile);
            if (tile == from.tile) tc::wait_for_dependency();   // the first kernel's image
            if (count == 0) continue;
            ok = tc::mbar_wait(low_done, (seg & 1) ^ 1, s_abort, &g_lora_status, kWaitAcc);   // nothing reads s_low any more
            if (!ok) break;
            if (tc::elect_one()) {
                tc::mbar_expect_tx(low_full, low_bytes);
                tc::bulk_load(s_low, p.image + (int64_t)tile * low_bytes, low_bytes, low_full);
            }
            __syncwarp();
            ok = tc::mbar_wait(low_full, seg & 1, s_abort, &g_lora_status, kWaitLow);
            ++seg;
            const int products = (end - begin) * count;
            for (int i = 0; i < products && ok; ++i, ++n) {
                const uint32_t buf = n & 1;
                ok = tc::mbar_wait(&acc_empty[buf], (n >> 1 & 1) ^ 1, s_abort, &g_lora_status, kWaitAccFree);
                if (!ok) break;
                for (int k = 0; k < k_steps; k += 4, br.next(plan.b_stages)) {
                    ok = tc::mbar_wait(&b_full[br.at], br.round, s_abort, &g_lora_status, kWaitFull);
                    if (!ok) break;
                    tc::fence_after();
                    if (tc::elect_one()) {
                        const uint32_t d = tmem + buf * kStep, to_lo = plan.blocks * (kTileBytes >> 4);
                        const uint32_t da = tc::desc_lo(s_low) + (k >> 2) * (kTileBytes >> 4), db = tc::desc_lo(s_b + br.at * b_bytes);
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (k + u < k_steps) {
                                tc::mma_16bit(d, da + 2 * u, db + 2 * u, desc, k + u > 0);
                                tc::mma_16bit(d, da + to_lo + 2 * u, db + 2 * u, desc, 1);
                            }
                        tc::commit(&b_empty[br.at]);
                        if (k + 4 >= k_steps) {
                            tc::commit(&acc_full[buf]);
                            if (i + 1 == products) tc::commit(low_done);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok) {
            if (tc::elect_one()) tc::commit(drain);
            __syncwarp();
            tc::mbar_drain(drain, 0);
            if (seg > 0) tc::mbar_drain(low_full, (seg - 1) & 1);
        }
    } else if (warp == 11) {
        // stores in the units' order; a stage is handed back one store later, when its own has read it
        tc::wait_for_dependency();   // (a CTA without a share waits here, too: this grid ends behind those that it hangs on, whose tables are in a
                                     // workspace that the next kernel may have been given)
        tc::Ring yr;
        int before = -1;
        bool ok = true;
        for (int tile = from.tile; tile <= tile1 && ok; ++tile) {
            const int begin = begin_of(tile), end = end_of(tile);
            if (in_place && tile_count(tile) == 0) continue;
            for (int unit = begin * kU; unit < end * kU; ++unit, yr.next(plan.y_stages)) {
                ok = tc::mbar_wait(&y_done[yr.at], yr.round, s_abort, &g_lora_status, kWaitDone);
                if (!ok) break;
                if (lane == 0) {
                    tc::tma_store_2d(&map_out, s_y + yr.at * kTileBytes, unit * 64, tile * kTile);
                    tc::tma_store_commit();
                    tc::tma_store_wait_read<1>();
                    if (before >= 0) tc::mbar_arrive(&y_empty[before]);
                }
                __syncwarp();
                before = yr.at;
            }
        }
        if (lane == 0) tc::tma_store_wait_read<0>();
        __syncwarp();
    } else {
        const uint32_t group = (warp - 2) >> 2;
        const int quarter = warp & 3, r_in_tile = quarter * 32 + lane;
        const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
        tc::Ring yr;                    // the step's first unit
        uint32_t n = 0;                 // accumulators so far
        uint32_t odd = 0;               // the parity of the step's first unit: which group takes it
        bool ok = true;
        for (int tile = from.tile; tile <= tile1 && ok; ++tile) {
            const int begin = begin_of(tile), end = end_of(tile);
            const int count = tile_count(tile);
            const int mine = __ldcg(p.slot128 + (int64_t)tile * kTile + r_in_tile);
            if (tile == from.tile) tc::wait_for_dependency();   // the first kernel's factors
            if (count == 0 && in_place) continue;
            const float factor = mine >= 0 ? __ldcg(p.factor + (int64_t)tile * kTile + r_in_tile) : 0.0f;
            for (int step = begin; step < end && ok; ++step) {
                for (int j = 0; j < count && ok; ++j, ++n) {
                    const uint32_t buf = n & 1;
                    ok = tc::mbar_wait(&acc_full[buf], n >> 1 & 1, s_abort, &g_lora_status, kWaitAcc);
                    if (!ok) break;
                    tc::fence_after();
                    if (__any_sync(0xffffffffu, mine == j)) {
                        tc::Ring r = yr;
#pragma unroll 1
                        for (uint32_t u = 0; u < kU; ++u, r.next(plan.y_stages)) {
                            if (((u + odd) & 1) != group) continue;
                            uint8_t* mine_y = s_y + r.at * kTileBytes + r_in_tile * 128;
                            uint32_t v[4][16];
#pragma unroll
                            for (int c = 0; c < 4; ++c) tc::ld16(acc + buf * kStep + u * 64 + 16 * c, v[c]);
                            tc::wait_ld();
                            ok = ok && tc::mbar_wait(&y_full[r.at], r.round, s_abort, &g_lora_status, kWaitY);
                            if (ok && mine == j) {
                                // (all of y's row is read before any of it is written: nothing orders the eight chunks)
                                Raw8<T> raw[8];
#pragma unroll
                                for (int c = 0; c < 8; ++c) raw[c].u = *reinterpret_cast<const uint4*>(mine_y + ((c ^ (r_in_tile & 7)) << 4));
#pragma unroll
                                for (int c = 0; c < 8; ++c) {
                                    float f[8];
                                    unpack8(raw[c], f);
#pragma unroll
                                    for (int i = 0; i < 8; ++i) f[i] = fmaf(factor, __uint_as_float(v[c >> 1][8 * (c & 1) + i]), f[i]);
                                    raw[c].u = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
                                }
#pragma unroll
                                for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(mine_y + ((c ^ (r_in_tile & 7)) << 4)) = raw[c].u;
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
                for (uint32_t u = 0; u < kU; ++u, yr.next(plan.y_stages)) {
                    if (((u + odd) & 1) != group) continue;
                    ok = ok && tc::mbar_wait(&y_full[yr.at], yr.round, s_abort, &g_lora_status, kWaitY);
                    if (ok && lane == 0) tc::mbar_arrive(&y_done[yr.at]);
                }
                odd ^= kU & 1;
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, kExpandColumns);
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

// Whether a call takes the kernel with a cluster per row.  Its time goes with rows x rank x (K + N), the adapters' elements
// that it reads from L2 (32 us at 67 M elements), that of the tiled kernels with the number of adapters that meet in a tile,
// which only the device knows: 64 rows of 16 adapters, rank 32, 4096 -> 14336: 17 us against 64 (one adapter: 20); 128
// rows 32 against 74 (21); 512 rows, rank 16, 4096 -> 4096: 37 against 91 (21).
bool few_rows(int64_t rows, int64_t K, int64_t N, int64_t R) { return rows <= 512 && rows * R * (K + N) <= 80000000; }

// What keeps tile coordinates, grids and the number of K steps within 32 bits.
constexpr int64_t kMostRows = 1 << 27, kMostColumns = 1 << 24;
bool units_fit(int64_t rows, int64_t K) { return ceil_div(rows, kShrinkRows) * ceil_div(K, 64) <= 0x3fffffff; }

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

ShrinkPlan shrink_plan(int64_t rows, int64_t K, int64_t R) {
    ShrinkPlan s{};
    s.k_tiles = (int)ceil_div(K, 64);
    s.halves = R > kTile ? 2 : 1;
    s.blocks = (int)ceil_div(R, 64);
    s.tiles = (int)ceil_div(rows, kShrinkRows);
    const int64_t most = ceil_div((int64_t)s.tiles * s.k_tiles, 4);   // at least four steps of K for a CTA
    s.ctas = (int)(most < sm_count() ? most : sm_count());
    const int a_bytes = s.halves * kTileBytes, rest = 1024 + 32 * 8 + 16 + 2 * (int)(sizeof(TileList) + sizeof(Place)) + 16;
    s.x_stages = (kSmemMost - rest - a_bytes) / (kXBytes + a_bytes);
    s.a_stages = s.x_stages + 1;
    s.smem = rest + s.x_stages * kXBytes + s.a_stages * a_bytes;
    return s;
}

// Where the parts of the workspace lie.
struct Workspace {
    int64_t factor, partial, lists, tables, bytes;   // (the image is at 0)
};
Workspace workspace_of(const ShrinkPlan& s, int64_t rows, int64_t R) {
    Workspace w{};
    w.factor = (int64_t)s.tiles * (kShrinkRows / kTile) * 2 * s.blocks * kTileBytes;
    w.partial = w.factor + round_up(rows * 4, 128);
    w.lists = w.partial + (int64_t)(s.ctas + s.tiles) * kShrinkRows * R * 4;
    w.tables = w.lists + (int64_t)s.tiles * (int64_t)sizeof(TileList);
    w.bytes = w.tables + (int64_t)s.tiles * (5 * 4 + kShrinkRows * (4 + 2));
    return w;
}

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return CK_OK;
    (void)cudaGetLastError();
    CK_FAIL((int)e, "lora_add (%s): %s", what, cudaGetErrorString(e));
}

// A launch; `chained`: its beginning may run beside the end of the kernel before it (wait_for_dependency()).
struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = {};
    Launch(unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, bool chained) {
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = chained ? 1 : 0;
    }
};

template <typename T, int kU>
int launch_expand(const LoraArgs& p, cudaStream_t stream) {
    constexpr int kStep = kU * 64, b_bytes = kStep * 128;
    ExpandPlan e{};
    e.steps = (int)ceil_div(p.N, kStep);
    e.tiles = (int)ceil_div(p.rows, kTile);
    e.k_steps = (int)ceil_div(p.R, 16);
    const int64_t items = (int64_t)e.steps * e.tiles;
    e.blocks = (int)ceil_div(p.R, 64);
    const int rest = 1024 + 64 * 8 + kTile * 4 + 2 * (int)sizeof(Place) + 16;
    // The image, a stage of B and four units of y (their number is even, so that a stage always serves
    // the same group of epilogue warps; a group that waited for a stage whose last load it had not seen might mistake that
    // one's end for its own); then, as far as there is room, six units of y, B for two steps, eight units of y.
    // (16384 x 8192, rank 128: six units with B for one step, 1 1/2 and 2: 227, 210 and 204 us; four units and two steps 214.)
    e.b_stages = 1;
    e.y_stages = 4;
    int room = kSmemMost - rest - 2 * e.blocks * kTileBytes - b_bytes - e.y_stages * kTileBytes;
    if (room < 0) CK_FAIL(CK_ERR_SHAPE, "lora_add: rank %lld does not fit", (long long)p.R);
    auto more_y = [&](int most) { while (e.y_stages < most && room >= 2 * kTileBytes) { e.y_stages += 2; room -= 2 * kTileBytes; } };
    more_y(6);
    while (e.b_stages < 2 * e.blocks + 1 && room >= b_bytes) { ++e.b_stages; room -= b_bytes; }
    more_y(8);
    e.smem = kSmemMost - room;
    CUtensorMap map_b, map_y, map_out;
    const int64_t bd[3] = {p.R, p.N, p.L}, bs[2] = {p.R * 2, p.N * p.R * 2};
    const int64_t yd[2] = {p.N, p.rows}, ys[1] = {p.y_stride * 2}, os[1] = {p.out_stride * 2};
    if (!tc::make_map_16bit(&map_b, p.b, 3, bd, bs, kStep) || !tc::make_map_16bit(&map_y, p.y, 2, yd, ys, kTile) ||
        !tc::make_map_16bit(&map_out, p.out, 2, yd, os, kTile))
        CK_FAIL(CK_ERR_UNSUPPORTED, "lora_add: a tensor map could not be encoded");
    auto kernel = lora_expand_kernel<T, kU>;
    const int rc = opt_in(kernel, kU + (Elem<T>::code == CK_BF16 ? 0 : 4) - 1);
    if (rc != CK_OK) return rc;
    Launch l((unsigned)(items < sm_count() ? items : sm_count()), kExpandThreads, e.smem, stream, true);
    return launched(cudaLaunchKernelEx(&l.cfg, kernel, map_b, map_y, map_out, p, e), "expand");
}

template <typename T>
int launch_many(LoraArgs p, uint8_t* workspace, cudaStream_t stream) {
    const ShrinkPlan s = shrink_plan(p.rows, p.K, p.R);
    const Workspace w = workspace_of(s, p.rows, p.R);
    p.image = workspace;
    p.factor = reinterpret_cast<float*>(workspace + w.factor);
    p.partial = reinterpret_cast<float*>(workspace + w.partial);
    p.asked128 = reinterpret_cast<int*>(workspace + w.tables);
    p.asked256 = p.asked128 + 2 * s.tiles;
    p.first_block = p.asked256 + s.tiles;
    p.last_block = p.first_block + s.tiles;
    p.list128 = p.last_block + s.tiles;
    p.slot128 = reinterpret_cast<int16_t*>(p.list128 + (int64_t)s.tiles * kShrinkRows);
    p.list256 = reinterpret_cast<TileList*>(workspace + w.lists);
    CUtensorMap map_x, map_a;
    const int64_t xd[2] = {p.K, p.rows}, xs[1] = {p.x_stride * 2};
    const int64_t ad[3] = {p.K, p.R, p.L}, as[2] = {p.K * 2, p.R * p.K * 2};
    if (!tc::make_map_16bit(&map_x, p.x, 2, xd, xs, kShrinkRows) || !tc::make_map_16bit(&map_a, p.a, 3, ad, as, (int)p.R))
        CK_FAIL(CK_ERR_UNSUPPORTED, "lora_add: a tensor map could not be encoded");
    int rc = opt_in(lora_shrink_kernel<T>, Elem<T>::code == CK_BF16);
    if (rc != CK_OK) return rc;
    Launch count((unsigned)s.tiles, 96, 0, stream, false);
    rc = launched(cudaLaunchKernelEx(&count.cfg, lora_count_kernel, p), "count");
    if (rc != CK_OK) return rc;
    Launch shrink((unsigned)s.ctas, kShrinkThreads, s.smem, stream, true);
    rc = launched(cudaLaunchKernelEx(&shrink.cfg, lora_shrink_kernel<T>, map_x, map_a, p, s), "shrink");
    if (rc != CK_OK) return rc;
    Launch join((unsigned)ceil_div(p.rows, kJoinThreads / 8), kJoinThreads, 0, stream, true);
    rc = launched(cudaLaunchKernelEx(&join.cfg, lora_join_kernel<T>, p, s), "join");
    if (rc != CK_OK) return rc;
    return ceil_div(p.rows, kTile) * ceil_div(p.N, 128) >= sm_count() ? launch_expand<T, 2>(p, stream) : launch_expand<T, 1>(p, stream);
}

}  // namespace
}  // namespace ck

extern "C" int64_t ck_lora_workspace_bytes(int64_t rows, int64_t K, int64_t N, int64_t rank) {
    using namespace ck;
    if (rows <= 0 || rows > kMostRows || K <= 0 || K > kMostColumns || N <= 0 || N > kMostColumns || rank <= 0 || rank > kMaxRank) return 0;   // (refused)
    if (few_rows(rows, K, N, rank) || !units_fit(rows, K)) return 0;
    return workspace_of(shrink_plan(rows, K, rank), rows, rank).bytes;
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
    if (rows <= 0 || rows > kMostRows || K <= 0 || K > kMostColumns || N <= 0 || N > kMostColumns || adapters <= 0 || adapters > 0x7fffffff ||
        K % 8 != 0 || N % 8 != 0 || rows_per_id <= 0 || x_row_stride < K || y_row_stride < N || out_row_stride < N)
        CK_FAIL(CK_ERR_SHAPE, "lora_add: bad shape rows=%lld K=%lld N=%lld adapters=%lld (K and N multiples of 8)", (long long)rows,
                (long long)K, (long long)N, (long long)adapters);
    if (!units_fit(rows, K))
        CK_FAIL(CK_ERR_SHAPE, "lora_add: %lld rows of %lld are too many", (long long)rows, (long long)K);
    if (rank <= 0 || rank % 8 != 0 || rank > kMaxRank) CK_FAIL(CK_ERR_SHAPE, "lora_add: rank %lld (a multiple of 8, at most %d)", (long long)rank, kMaxRank);
    if (!aligned16(y) || !aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(out) || ((x_row_stride | y_row_stride | out_row_stride) & 7))
        CK_FAIL(CK_ERR_ALIGN, "lora_add: tensors and row strides must be 16-byte aligned");
    // A row's columns are written by several CTAs and other rows by others, in no order, so what they read stays, but for y in its own
    // place and x's same row (every kernel is done with a row of x before it writes that row).
    const Memory written{out, rows, out_row_stride * 2, N * 2}, added{y, rows, y_row_stride * 2, N * 2}, taken{x, rows, x_row_stride * 2, K * 2};
    if (overlap(written, added) && !same_place(written, added)) CK_FAIL(CK_ERR_UNSUPPORTED, "lora_add: out overlaps y and is not y");
    if ((overlap(written, taken) && !row_by_row(written, taken)) || overlap(written, memory_of(a, adapters * rank * K * 2)) ||
        overlap(written, memory_of(b, adapters * rank * N * 2)) || overlap(written, memory_of(scales, adapters * 4)) ||
        overlap(written, memory_of(ids, ceil_div(rows, rows_per_id) * (ids_64bit ? 8 : 4))))
        CK_FAIL(CK_ERR_UNSUPPORTED, "lora_add: out overlaps an input");
    const LoraArgs p{y, x, a, b, ids, scales, out, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, rows, K, N, rank, adapters, y_row_stride, x_row_stride, out_row_stride, rows_per_id, ids_64bit};
    if (few_rows(rows, K, N, rank)) {
        const dim3 grid(kFewCluster, (unsigned)rows);
        if (dtype_code == CK_BF16) lora_few_kernel<__nv_bfloat16><<<grid, kFewThreads, 0, stream>>>(p);
        else lora_few_kernel<__half><<<grid, kFewThreads, 0, stream>>>(p);
        return launch_status("lora_add");
    }
    if (!workspace) CK_FAIL(CK_ERR_NULL, "lora_add: a workspace of ck_lora_workspace_bytes() is needed");
    if (!aligned16(workspace)) CK_FAIL(CK_ERR_ALIGN, "lora_add: the workspace must be 16-byte aligned");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    return dtype_code == CK_BF16 ? launch_many<__nv_bfloat16>(p, ws, stream) : launch_many<__half>(p, ws, stream);
}
