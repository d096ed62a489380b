// Rotary embedding by positions of several axes (time, height, width) for sm_100a, without a table.
//
// Pair p of a head belongs to one axis; at token n it turns by  angle = position[n, axis(p)] * freqs[p]:
//   (a, b) -> (a cos - b sin, a sin + b cos),  (a, b) = (x[2p], x[2p+1])  or, split-half,  (x[p], x[p + P])
// with P pairs in all; elements from 2P on pass through.  freqs is in radians per unit of position, in 64 bits:
// at a position of 10^6 a product in 32 bits is already 0.03 rad off.  The turn is reduced to [-1/2, 1/2] in
// 64 bits and rounded to fp32 for the sine and cosine, which then take up what the rounding left (to first order: error
// against 64 bits 3.6e-8 instead of 4.7e-8, at no cost that shows), at any position; the rotation is in fp32 with one rounding to x's type.  The inverse rotation (the
// transpose, which is the gradient's) changes the sine's sign.
//
// Bound by HBM: q and k are read and written once (positions are a few bytes a token; rope.cu reads 4 fp32 per
// pair of table instead); 25037 tokens x 80 heads x 128 in 162.5 us back to back, 6.31 TB/s, 98 % of the copy rate.  A thread owns 4 pairs of one token (8 with split-half), computes their sines and cosines
// once and walks heads of q and k with them, moving 16 bytes of 16-bit data a step.
#include "ck_common.cuh"

namespace ck {
namespace {

constexpr int kMaxAxes = 8;
constexpr int kThreads = 128;
enum PosType { kPosF32 = 0, kPosF64 = 1, kPosI32 = 2, kPosI64 = 3 };

struct RopeAxesParams {
    const void* x[2];          // q, k (k may be null)
    void* o[2];                // contiguous in the order of x's dimensions
    const void* pos;
    const double* freqs;       // [P]
    int64_t sx[2][4];          // element strides of batch, token, head, element
    int64_t so[2][3];          // output strides of batch, token, head
    int64_t sp[3];             // position strides of batch, token, axis
    int64_t batch, tokens;
    int heads[2];
    int D, P, n_axes, pos_type;
    int axis_end[kMaxAxes];    // first pair behind each axis' pairs
    int n_vec;                 // work items per token and head chunk
    int chunk, n_chunks;       // heads (of q, then k) one thread walks
    float sign;                // -1: inverse
};

__device__ __forceinline__ double position(const RopeAxesParams& p, int64_t off) {
    switch (p.pos_type) {
    case kPosF32: return (double)__ldg(static_cast<const float*>(p.pos) + off);
    case kPosF64: return __ldg(static_cast<const double*>(p.pos) + off);
    case kPosI32: return (double)__ldg(static_cast<const int*>(p.pos) + off);
    default: return (double)__ldg(static_cast<const long long*>(p.pos) + off);
    }
}

// Cosine and sine of pair `pair` at the token whose positions start at `off`.
__device__ __forceinline__ float2 pair_turn(const RopeAxesParams& p, int64_t off, int pair) {
    int axis = 0;
#pragma unroll
    for (int i = 0; i < kMaxAxes - 1; ++i)
        if (i < p.n_axes - 1 && pair >= p.axis_end[i]) axis = i + 1;
    const double turns = position(p, off + axis * p.sp[2]) * (__ldg(p.freqs + pair) * 0.15915494309189533577 /* 1 / 2 pi */);
    const double half_turns = 2.0 * (turns - rint(turns));
    const float near = (float)half_turns, rest = (float)(half_turns - (double)near) * 3.14159265f;   // (at most 2^-25 half turns)
    float s, c;
    sincospif(near, &s, &c);
    return make_float2(fmaf(-s, rest, c), p.sign * fmaf(c, rest, s));
}

__device__ __forceinline__ void rotate(float2 t, float a, float b, float& oa, float& ob) {
    oa = fmaf(a, t.x, -__fmul_rn(b, t.y));
    ob = fmaf(a, t.y, __fmul_rn(b, t.x));
}

// Where head `head` (q's heads first, then k's) of the item starts in the input and the output.
template <typename T>
__device__ __forceinline__ void head_at(const RopeAxesParams& p, int64_t b, int64_t n, int head, const T*& src, T*& dst) {
    const int which = head < p.heads[0] ? 0 : 1;
    const int64_t h = which ? head - p.heads[0] : head;
    src = static_cast<const T*>(p.x[which]) + b * p.sx[which][0] + n * p.sx[which][1] + h * p.sx[which][2];
    dst = static_cast<T*>(p.o[which]) + b * p.so[which][0] + n * p.so[which][1] + h * p.so[which][2];
}

// Two pairs: (a0, a1) cos - (b0, b1) sin and (a0, a1) sin + (b0, b1) cos; 16-bit types with sm_100's packed fp32 instructions.
// (fp32 has half as many elements a byte and instructions to spare; packed it took 20.2 us for 3 x 1377 x 25 heads of 80, not 17.3.)
template <typename T>
__device__ __forceinline__ void rotate2(float2 c, float2 s, float2& a, float2& b) {
    float2 oa;
    if (sizeof(T) == 4) {
        const float2 ia = a, ib = b;
        rotate(make_float2(c.x, s.x), ia.x, ib.x, oa.x, b.x);
        rotate(make_float2(c.y, s.y), ia.y, ib.y, oa.y, b.y);
    } else {
        oa = __ffma2_rn(b, make_float2(-s.x, -s.y), __fmul2_rn(a, c));
        b = __ffma2_rn(b, c, __fmul2_rn(a, s));
    }
    a = oa;
}

// Vectors of 8 elements: unit stride, D (and, split-half, P) a multiple of 8, 16-byte aligned rows.  The loop over heads is
// kept to a few instructions an element (pointers that step by the head's stride, packed arithmetic): with 64-bit
// offsets worked out for every head it took 140 instructions a vector, 80 % of the issue slots at full clock, and was
// no longer bound by HBM where the clock is lower.
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kThreads) rope_axes_vec_kernel(const RopeAxesParams p) {
    constexpr int kPairs = kSplit ? 8 : 4;
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t site = item / p.n_vec;
    const int v = (int)(item - site * p.n_vec);
    if (site >= p.tokens) return;
    const int64_t b = blockIdx.y / p.n_chunks;
    const int h0 = (int)(blockIdx.y % p.n_chunks) * p.chunk;
    const int h1 = min(h0 + p.chunk, p.heads[0] + p.heads[1]);

    // columns of this thread: one vector (interleaved), or the two vectors of a split-half item; behind the
    // rotated part a split-half item is two neighbouring vectors that pass through
    const int turning = kSplit ? p.P / 8 : (2 * p.P + 7) / 8;
    const bool rotates = v < turning;
    const int lo = kSplit && !rotates ? 2 * p.P + (v - turning) * 16 : v * 8;
    const int apart = kSplit ? (rotates ? p.P : 8) : 0;
    const bool second = kSplit && lo + apart < p.D;
    const bool whole = kSplit || (v + 1) * 4 <= p.P;   // (interleaved: all four pairs turn)
    float2 c[kPairs / 2], s[kPairs / 2];               // of pairs 2 i and 2 i + 1
    if (rotates) {
        const int64_t off = b * p.sp[0] + site * p.sp[1];
#pragma unroll
        for (int i = 0; i < kPairs / 2; ++i) {
            const int pair = v * kPairs + 2 * i;
            const float2 t0 = pair < p.P ? pair_turn(p, off, pair) : make_float2(1.0f, 0.0f);
            const float2 t1 = pair + 1 < p.P ? pair_turn(p, off, pair + 1) : make_float2(1.0f, 0.0f);
            c[i] = make_float2(t0.x, t1.x);
            s[i] = make_float2(t0.y, t1.y);
        }
    }
    constexpr int kBatch = kSplit ? 2 : 4;
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {          // q's heads of the chunk, then k's
        const int first = which ? p.heads[0] : 0;
        const int from = max(h0, first) - first, n = min(h1, first + p.heads[which]) - first - from;
        const int64_t step_in = p.sx[which][2], step_out = p.so[which][2];
        const T* src = static_cast<const T*>(p.x[which]) + b * p.sx[which][0] + site * p.sx[which][1] + from * step_in + lo;
        T* dst = static_cast<T*>(p.o[which]) + b * p.so[which][0] + site * p.so[which][1] + from * step_out + lo;
        auto turn = [&](Raw8<T>& ra, Raw8<T>& rb, T* out) {
            float x[8], y[8];
            unpack8(ra, x);
            if (kSplit) {
                if (second) unpack8(rb, y);
                if (rotates) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float2 e = make_float2(x[2 * i], x[2 * i + 1]), f = make_float2(y[2 * i], y[2 * i + 1]);
                        rotate2<T>(c[i], s[i], e, f);
                        x[2 * i] = e.x; x[2 * i + 1] = e.y;
                        y[2 * i] = f.x; y[2 * i + 1] = f.y;
                    }
                }
                store8<T>(out, x);
                if (second) store8<T>(out + apart, y);
            } else {
                if (rotates) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float2 e = make_float2(x[4 * i], x[4 * i + 2]), f = make_float2(x[4 * i + 1], x[4 * i + 3]);
                        rotate2<T>(c[i], s[i], e, f);
                        if (whole || v * 4 + 2 * i < p.P) { x[4 * i] = e.x; x[4 * i + 1] = f.x; }
                        if (whole || v * 4 + 2 * i + 1 < p.P) { x[4 * i + 2] = e.y; x[4 * i + 3] = f.y; }
                    }
                }
                store8<T>(out, x);
            }
        };
        int h = 0;
#pragma unroll 1
        for (; h + kBatch <= n; h += kBatch, src += kBatch * step_in, dst += kBatch * step_out) {
            Raw8<T> ra[kBatch], rb[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                ra[i] = load_raw8<T>(src + i * step_in);
                if (second) rb[i] = load_raw8<T>(src + i * step_in + apart);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) turn(ra[i], rb[i], dst + i * step_out);
        }
#pragma unroll 1
        for (; h < n; ++h, src += step_in, dst += step_out) {
            Raw8<T> ra = load_raw8<T>(src), rb = ra;
            if (second) rb = load_raw8<T>(src + apart);
            turn(ra, rb, dst);
        }
    }
}

// Any strides, any even D: one pair per thread and head; a thread behind the pairs copies two elements.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_axes_generic_kernel(const RopeAxesParams p, const bool split) {
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t site = item / p.n_vec;
    const int pair = (int)(item - site * p.n_vec);
    if (site >= p.tokens) return;
    const int64_t b = blockIdx.y / p.n_chunks;
    const int h0 = (int)(blockIdx.y % p.n_chunks) * p.chunk;
    const int h1 = min(h0 + p.chunk, p.heads[0] + p.heads[1]);
    const bool rotates = pair < p.P;
    const int ia = split && rotates ? pair : 2 * pair, ib = split && rotates ? pair + p.P : 2 * pair + 1;
    const float2 t = rotates ? pair_turn(p, b * p.sp[0] + site * p.sp[1], pair) : make_float2(1.0f, 0.0f);
    for (int h = h0; h < h1; ++h) {
        const T* src;
        T* dst;
        head_at<T>(p, b, site, h, src, dst);
        const int64_t se = p.sx[h < p.heads[0] ? 0 : 1][3];
        const T a = src[ia * se], c = src[ib * se];
        if (rotates) {
            float oa, oc;
            rotate(t, Elem<T>::to_f32(a), Elem<T>::to_f32(c), oa, oc);
            dst[ia] = Elem<T>::from_f32(oa);
            dst[ib] = Elem<T>::from_f32(oc);
        } else {
            dst[ia] = a;
            dst[ib] = c;
        }
    }
}

template <typename T>
int launch(RopeAxesParams p, bool split, bool vec, cudaStream_t stream) {
    p.n_vec = vec ? (split ? p.P / 8 + (int)ceil_div(p.D - 2 * p.P, 16) : p.D / 8) : p.D / 2;
    const int heads = p.heads[0] + p.heads[1];
    // A thread walks at most 16 heads: enough to make the sines cheap, few enough for the last CTAs to end together
    // (25037 tokens x 80 heads: 159 us; 80 heads a thread 177, 10 heads 173), and fewer while an SM has less than 768
    // threads (3 x 1377 x 25: 17 us with 5 heads a thread, 22.2 with all; one token: 4.1 us with one, 4.9 with four).
    const int64_t gx = ceil_div(p.tokens * p.n_vec, kThreads);
    if (gx > 0x7fffffff) CK_FAIL(CK_ERR_SHAPE, "apply_rope_axes: %lld tokens are more than a grid holds", (long long)p.tokens);
    const int64_t sites = p.batch * p.tokens * p.n_vec;
    int64_t chunks = ceil_div(148LL * 768, sites);
    if (chunks > heads) chunks = heads;
    if (chunks < ceil_div(heads, 16)) chunks = ceil_div(heads, 16);
    if (chunks > 65535 / p.batch) chunks = 65535 / p.batch;   // (batch x chunks is a grid dimension)
    if (chunks < 1) chunks = 1;
    p.chunk = (int)ceil_div(heads, chunks);
    p.n_chunks = (int)ceil_div(heads, p.chunk);
    const dim3 grid((unsigned)gx, (unsigned)(p.batch * p.n_chunks));
    if (!vec) rope_axes_generic_kernel<T><<<grid, kThreads, 0, stream>>>(p, split);
    else if (split) rope_axes_vec_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
    else rope_axes_vec_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
    return launch_status("apply_rope_axes");
}

}  // namespace
}  // namespace ck

extern "C" int launch_apply_rope_axes_kernel(const void* xq, const void* xk, const void* positions, const double* freqs,
                                             void* xq_out, void* xk_out, const int64_t* strides, int64_t batch, int64_t tokens,
                                             int64_t heads_q, int64_t heads_k, int64_t head_dim, const int32_t* axis_pairs,
                                             int n_axes, int dtype_code, int positions_code, bool tokens_first, bool split_half, bool inverse,
                                             cudaStream_t stream) {
    using namespace ck;
    if (!xq || !positions || !freqs || !xq_out || !strides || !axis_pairs) CK_FAIL(CK_ERR_NULL, "apply_rope_axes: null pointer");
    if ((xk == nullptr) != (xk_out == nullptr) || (xk == nullptr) != (heads_k == 0))
        CK_FAIL(CK_ERR_NULL, "apply_rope_axes: xk, xk_out and heads_k must be given together");
    if (batch <= 0 || batch > 65535 || tokens <= 0 || tokens > (1LL << 40) || heads_q <= 0 || heads_k < 0 || heads_q > 65535 || heads_k > 65535 || head_dim <= 0 ||
        head_dim % 2 != 0 || head_dim > 65536)
        CK_FAIL(CK_ERR_SHAPE, "apply_rope_axes: bad shape batch=%lld tokens=%lld heads=%lld/%lld head_dim=%lld (even)", (long long)batch,
                (long long)tokens, (long long)heads_q, (long long)heads_k, (long long)head_dim);
    if (n_axes < 1 || n_axes > kMaxAxes) CK_FAIL(CK_ERR_SHAPE, "apply_rope_axes: %d axes (1 to %d)", n_axes, kMaxAxes);
    if (positions_code < kPosF32 || positions_code > kPosI64) CK_FAIL(CK_ERR_DTYPE, "apply_rope_axes: positions type code %d", positions_code);
    RopeAxesParams p{};
    int64_t pairs = 0;
    for (int i = 0; i < n_axes; ++i) {
        if (axis_pairs[i] <= 0) CK_FAIL(CK_ERR_SHAPE, "apply_rope_axes: axis %d has %d pairs", i, (int)axis_pairs[i]);
        pairs += axis_pairs[i];
        if (2 * pairs > head_dim) CK_FAIL(CK_ERR_SHAPE, "apply_rope_axes: the axes turn more than %lld elements", (long long)head_dim);
        p.axis_end[i] = (int)pairs;
    }
    p.x[0] = xq; p.x[1] = xk; p.o[0] = xq_out; p.o[1] = xk_out;
    p.pos = positions; p.freqs = freqs;
    // strides: q (batch, token, head, element), k (the same), positions (batch, token, axis)
    for (int i = 0; i < 4; ++i) { p.sx[0][i] = strides[i]; p.sx[1][i] = strides[4 + i]; }
    for (int i = 0; i < 3; ++i) p.sp[i] = strides[8 + i];
    const int64_t heads[2] = {heads_q, heads_k};
    for (int w = 0; w < 2; ++w) {
        p.so[w][0] = heads[w] * tokens * head_dim;
        p.so[w][1] = tokens_first ? heads[w] * head_dim : head_dim;
        p.so[w][2] = tokens_first ? head_dim : tokens * head_dim;
    }
    p.batch = batch; p.tokens = tokens; p.heads[0] = (int)heads_q; p.heads[1] = (int)heads_k;
    p.D = (int)head_dim; p.P = (int)pairs; p.n_axes = n_axes; p.pos_type = positions_code;
    p.sign = inverse ? -1.0f : 1.0f;
    bool vec = head_dim % 8 == 0 && (!split_half || pairs % 8 == 0);
    for (int w = 0; w < (xk ? 2 : 1); ++w) {
        vec = vec && aligned16(p.x[w]) && aligned16(p.o[w]) && p.sx[w][3] == 1;
        for (int i = 0; i < 3; ++i) vec = vec && p.sx[w][i] % 8 == 0 && p.so[w][i] % 8 == 0;
    }
    switch (dtype_code) {
    case CK_F32: return launch<float>(p, split_half, vec, stream);
    case CK_F16: return launch<__half>(p, split_half, vec, stream);
    case CK_BF16: return launch<__nv_bfloat16>(p, split_half, vec, stream);
    default: CK_FAIL(CK_ERR_DTYPE, "apply_rope_axes: unsupported dtype code %d", dtype_code);
    }
}
