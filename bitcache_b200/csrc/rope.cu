// Per-head query/key norms with position rotation, alone (bc_qk_norm_rope) and
// on the way into a paged quantised cache (bc_append_qkv_paged).  sm_100a.
//
// For a head row x of head_dim elements at token position p:
//   y_i = (x_i * r) * w_i,  r = 1 / sqrt(sum(x^2) / head_dim + eps)     (norm; y = x without weights)
//   pairs (i, j) of the rotary_dim first elements (j = i + rotary_dim / 2, or
//   adjacent elements when interleaved), c = cos[p][pair], s = sin[p][pair]:
//   z_i = y_i c - y_j s,  z_j = y_j c + y_i s                            (rotation)
// Keys and values then become sign bits, mean |z| and INT4 residual codes
// (encode_core.cuh).
//
// Every product, sum, quotient and root below is rounded on its own (no
// contraction), sums run in the encoders' stride-halving tree order, and this
// file is compiled without fast-math, so an implementation in any framework
// that follows the same order gets the same planes bit for bit.  The encoders
// of encode.cu divide with fast-math as the reference does; their codes can
// differ from these by one where 7 r / absmax lies next to a rounding tie.
#include <cuda_bf16.h>

#include "encode_core.cuh"

namespace bc {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }

struct RopeArgs {
    bc_heads q, k, v;
    const int32_t* positions;
    const int32_t* seq_ids;  // append only
    bc_rope rope;
    void* q_out;
    void* k_out;  // bc_qk_norm_rope: rotated keys; append: rows as the cache holds them (k_hat), may be null
    void* v_out;  // append: v_hat, may be null
    bc_kv_planes K, V;
    bc_page_table pt;
    int64_t n_tokens;
    int n_seqs, n_heads, n_kv_heads;
    unsigned int* err;
};

// Cache row of token t for kv head h (h < 0: a query, which has none: 0), or -1
// where an index lies outside its range, which raises an error bit.
__device__ __forceinline__ int64_t append_row(const RopeArgs& a, int64_t t, int pos, int h) {
    const int seq = a.seq_ids[t];
    if (seq < 0 || seq >= a.n_seqs || pos >= (int64_t)a.pt.max_pages * a.pt.page_size) {
        raise_device_error(a.err, BC_DEVERR_INDEX);
        return -1;
    }
    if (h < 0) return 0;
    const int64_t slot = (int64_t)seq * a.n_kv_heads + h;
    const int pg = a.pt.pages[slot * a.pt.max_pages + pos / a.pt.page_size];
    if (pg < 0 || pg >= a.pt.n_pages) {
        raise_device_error(a.err, BC_DEVERR_PAGE);
        return -1;
    }
    return (int64_t)pg * a.pt.page_size + pos % a.pt.page_size;
}

// ---------------------------------------------------------------------------
// Any head_dim, rotary_dim, alignment: one warp per head row, lane l holds
// elements l + 32k; the row passes through shared memory for the pairs.
// ---------------------------------------------------------------------------
constexpr int kRopeWarps = 8;

template <int NW, typename T, typename O, bool APPEND, int RES>
__global__ void __launch_bounds__(kRopeWarps * 32) k_rope_rows(const RopeArgs a) {
    constexpr int D = 32 * NW;
    __shared__ float rows[kRopeWarps][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = a.n_heads + (APPEND ? 2 : 1) * a.n_kv_heads;
    const int64_t job = (int64_t)blockIdx.x * kRopeWarps + warp;
    if (job >= a.n_tokens * heads) return;
    const int64_t t = job / heads;
    int h = (int)(job - t * heads);
    const int kind = h < a.n_heads ? 0 : h < a.n_heads + a.n_kv_heads ? 1 : 2;
    h -= kind == 0 ? 0 : kind == 1 ? a.n_heads : a.n_heads + a.n_kv_heads;
    const bc_heads& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const T* src = reinterpret_cast<const T*>(in.data) + t * in.token_stride + (int64_t)h * in.head_stride;
    O* out = reinterpret_cast<O*>(kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out);
    if (out) out += (t * (kind == 0 ? a.n_heads : a.n_kv_heads) + h) * D;

    int pos = a.positions[t];
    if (a.rope.cos && pos >= a.rope.n_positions) {
        if (lane == 0) raise_device_error(a.err, BC_DEVERR_INDEX);
        pos = -1;
    }
    int64_t row = -1;
    if (APPEND && pos >= 0) {
        if (lane == 0) row = append_row(a, t, pos, kind == 0 ? -1 : h);
        row = __shfl_sync(0xffffffffu, row, 0);
    }
    if (pos < 0 || (APPEND && row < 0)) {  // padding
        if (out)
            for (int k = 0; k < NW; ++k) out[32 * k + lane] = from_f<O>(0.0f);
        return;
    }
    float x[NW];
#pragma unroll
    for (int k = 0; k < NW; ++k) x[k] = to_f<T>(src[32 * k + lane]);
    const float* w = kind == 0 ? a.rope.q_weight : kind == 1 ? a.rope.k_weight : nullptr;
    if (w) {
        float sq[NW];
#pragma unroll
        for (int k = 0; k < NW; ++k) sq[k] = __fmul_rn(x[k], x[k]);
        const float mean = __fdiv_rn(tree_abs_sum<NW>(sq), (float)D);  // squares: |.| changes nothing
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, a.rope.eps)));
#pragma unroll
        for (int k = 0; k < NW; ++k) x[k] = __fmul_rn(__fmul_rn(x[k], r), w[32 * k + lane]);
    }
    if (a.rope.cos && kind != 2) {
        float* y = rows[warp];
#pragma unroll
        for (int k = 0; k < NW; ++k) y[32 * k + lane] = x[k];
        __syncwarp();
        const int half = a.rope.rotary_dim / 2;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const int i = 32 * k + lane;
            if (i < 2 * half) {
                const int pair = a.rope.interleaved ? i >> 1 : (i < half ? i : i - half);
                const bool second = a.rope.interleaved ? (i & 1) : i >= half;
                const int j = a.rope.interleaved ? i ^ 1 : (second ? i - half : i + half);
                const float c = a.rope.cos[(int64_t)pos * half + pair], s = a.rope.sin[(int64_t)pos * half + pair];
                const float own = __fmul_rn(x[k], c), other = __fmul_rn(y[j], s);
                x[k] = second ? __fadd_rn(own, other) : __fsub_rn(own, other);
            }
        }
        __syncwarp();
    }
    if (!APPEND || kind == 0) {
#pragma unroll
        for (int k = 0; k < NW; ++k) out[32 * k + lane] = from_f<O>(x[k]);
        return;
    }
    encode_row_planes<NW, RES>(x, lane, D, kind == 1 ? a.K : a.V, row);
    if (out) {  // the row as the planes hold it
        const float mean_abs = tree_abs_sum<NW>(x) / (float)D;
        const float held = __half2float(__float2half(mean_abs));
        const float s = RES == BC_RES_FP16_SCALE ? held : mean_abs;
        float r[NW], lm = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            r[k] = x[k] - (x[k] >= 0.0f ? s : -s);
            lm = fmaxf(lm, fabsf(r[k]));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) lm = fmaxf(lm, __shfl_xor_sync(0xffffffffu, lm, off));
        const float inv = lm > 0.0f ? 7.0f / lm : 0.0f;
        const float rs = __half2float(__float2half(lm));
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float base = x[k] >= 0.0f ? held : -held;
            const int code = max(-7, min(7, __float2int_rn(__fmul_rn(r[k], inv))));
            out[32 * k + lane] =
                from_f<O>(RES == BC_RES_NONE ? base : __fadd_rn(base, __fmul_rn(__fdiv_rn((float)code, 7.0f), rs)));
        }
    }
}

// ---------------------------------------------------------------------------
// head_dim 64, 128, 256 on 16-byte boundaries: head_dim / 16 lanes a row, lane r
// with elements 8r .. 8r + 7 ("slot 0") and head_dim / 2 + 8r .. ("slot 1"), so a
// row is two 16-byte loads per lane, rotation pairs head_dim / 2 apart are a
// lane's own, and a sign byte and its nibble bytes are too.  A warp takes several
// heads of one token at a time (4 at 128), with the token's cosines and sines in
// registers.  The tree sums cost 10 shuffles for 4 rows here, 20 in the kernel above,
// whose 2-byte loads also keep too little in flight.  Norm and rotation alone are
// bound by HBM: 16384 tokens of 32 + 8 heads of 128, bf16, 72 us, 4.8 TB/s (the
// same rows through registers instead of the lanes' rings of copies: 117 us; in the
// kernel above 257).  The append is bound by the instructions that encode 16 of a
// token's 48 rows and, with two CTAs an SM, by their latency: 24 prompts of
// 512 to 1024 tokens, same heads, with k_hat and v_hat, 154 us, 3.2 TB/s (528 above).
// ---------------------------------------------------------------------------
template <int D>
struct Lanes {
    static constexpr int LPR = D / 16;   // lanes of a row
    static constexpr int ROWS = 32 / LPR;  // rows of a warp
};

// The encoders' tree: leaf t holds v_t, strides 128, 64, ..., 1.  p[j] is the sum
// over both slots already (the first stride).  Lanes halve the eight positions
// they are responsible for at each stride, then the positions meet.
template <int D>
__device__ __forceinline__ float group_tree(float (&p)[8], int lane) {
    constexpr int LPR = Lanes<D>::LPR;
    int n = 8;
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
        if (n > 1) {
            const bool up = lane & o;
            n >>= 1;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) {
                    const float give = up ? p[j] : p[j + n], keep = up ? p[j + n] : p[j];
                    p[j] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, o));
                }
        } else {
            p[0] = __fadd_rn(p[0], __shfl_xor_sync(0xffffffffu, p[0], o));
        }
    }
    if constexpr (LPR == 4) {  // lanes 2, 1 hold position bits 2, 1; bit 0 is local
#pragma unroll
        for (int o = 2; o > 0; o >>= 1)
#pragma unroll
            for (int j = 0; j < 2; ++j) p[j] = __fadd_rn(p[j], __shfl_xor_sync(0xffffffffu, p[j], o));
        return __fadd_rn(p[0], p[1]);
    } else {
#pragma unroll
        for (int o = LPR / 2; o > LPR / 16; o >>= 1) p[0] = __fadd_rn(p[0], __shfl_xor_sync(0xffffffffu, p[0], o));
        return p[0];
    }
}

// A lane's own ring of copies: `stages` ahead of use, without a register and
// without a barrier, since each lane reads back what it has asked for.
template <typename T>
struct Ring {
    static constexpr int UNITS = sizeof(T) == 4 ? 4 : 2;   // 16-byte units of a lane's 16 elements
    static constexpr int STAGES = sizeof(T) == 4 ? 3 : 4;
    static constexpr int WARP_B = STAGES * UNITS * 512;
};
__device__ __forceinline__ void copy16(uint8_t* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 read16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(p)) : "memory");
    return v;
}
// Slot y of the lane's 16 elements in a stage at `at` (the lane's first unit).
__device__ __forceinline__ void load8(const uint8_t* at, int y, __half, float (&x)[8]) {
    const uint4 v = read16(at + 512 * y);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const uint8_t* at, int y, __nv_bfloat16, float (&x)[8]) {
    const uint4 v = read16(at + 512 * y);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load8(const uint8_t* at, int y, float, float (&x)[8]) {
    const uint4 v = read16(at + 1024 * y), w = read16(at + 1024 * y + 512);
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    x[4] = __uint_as_float(w.x), x[5] = __uint_as_float(w.y), x[6] = __uint_as_float(w.z), x[7] = __uint_as_float(w.w);
}

// Two products at once, each rounded as alone.  Only for products of products: with a
// packed sum behind a packed product, results were seen to differ from those of
// operations rounded one by one.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 pair(const float (&x)[8], int j) { return make_float2(x[j], x[j + 1]); }
__device__ __forceinline__ void put(float (&x)[8], int j, float2 v) {
    x[j] = v.x;
    x[j + 1] = v.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename O>
__device__ __forceinline__ void store8(O* p, const float (&x)[8]) {
    if constexpr (sizeof(O) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], O{}), pack2(x[2], x[3], O{}), pack2(x[4], x[5], O{}),
                                                  pack2(x[6], x[7], O{}));
    }
}
__device__ __forceinline__ void load8f(const float* p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// 4 x 4 bytes transposed over lanes a = 0 .. 3: lane a gets byte a of each lane's word.
__device__ __forceinline__ uint32_t transpose4(uint32_t x, int a) {
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, 1);
    const uint32_t u = a & 1 ? __byte_perm(x, y, 0x3715) : __byte_perm(x, y, 0x6240);
    const uint32_t z = __shfl_xor_sync(0xffffffffu, u, 2);
    return a & 2 ? __byte_perm(u, z, 0x3276) : __byte_perm(u, z, 0x5410);
}

enum { kPairsNone = 0, kPairsHalf = 1, kPairsApart = 2, kPairsNext = 3 };  // head_dim / 2 apart, rotary_dim / 2 apart, adjacent

// APART: kPairsApart (twice the cosines, and shuffles); otherwise `style`.
template <int D, typename T, typename O, bool APPEND, bool APART>
__global__ void __launch_bounds__(kRopeWarps * 32, APPEND ? 2 : 3) k_rope_lanes(const RopeArgs a, int style, int per, int res) {
    constexpr int LPR = Lanes<D>::LPR, ROWS = Lanes<D>::ROWS;
    using R = Ring<T>;
    __shared__ __align__(16) uint8_t ring[kRopeWarps * R::WARP_B];
    const int lane = threadIdx.x & 31, r = lane % LPR, sub = lane / LPR;
    const int heads = a.n_heads + (APPEND ? 2 : 1) * a.n_kv_heads;
    const int groups = (heads + ROWS - 1) / ROWS, runs = (groups + per - 1) / per;
    const int64_t job = (int64_t)blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
    if (job >= a.n_tokens * runs) return;
    const int64_t t = job / runs;
    const int g0 = (int)(job - t * runs) * per, g1 = min(groups, g0 + per);
    uint8_t* mine = ring + (threadIdx.x >> 5) * R::WARP_B + lane * 16;

    // row g of this lane's: what it is, where it lies
    auto place = [&](int g, int& kind, int& h) {
        h = g * ROWS + sub;
        kind = h < a.n_heads ? 0 : h < a.n_heads + a.n_kv_heads ? 1 : 2;
        h -= kind == 0 ? 0 : kind == 1 ? a.n_heads : a.n_heads + a.n_kv_heads;
    };
    auto fetch = [&](int g) {
        if (g < g1 && g * ROWS + sub < heads) {
            int kind, h;
            place(g, kind, h);
            const bc_heads& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
            const T* src = reinterpret_cast<const T*>(in.data) + t * in.token_stride + h * in.head_stride + 8 * r;
            uint8_t* dst = mine + (g - g0) % R::STAGES * (R::UNITS * 512);
#pragma unroll
            for (int u = 0; u < R::UNITS / 2; ++u) {
                copy16(dst + 512 * u, reinterpret_cast<const uint8_t*>(src) + 16 * u);
                copy16(dst + 512 * (R::UNITS / 2 + u), reinterpret_cast<const uint8_t*>(src + D / 2) + 16 * u);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < R::STAGES; ++i) fetch(g0 + i);

    int pos = a.positions[t];
    bool bad = a.rope.cos && pos >= a.rope.n_positions;
    int seq = 0;
    if constexpr (APPEND) {
        seq = a.seq_ids[t];
        bad = bad || (pos >= 0 && (seq < 0 || seq >= a.n_seqs || pos >= (int64_t)a.pt.max_pages * a.pt.page_size));
    }
    if (bad) {
        if (lane == 0) raise_device_error(a.err, BC_DEVERR_INDEX);
        pos = -1;
    }
    const int half = a.rope.rotary_dim / 2;
    int page = 0, in_page = 0;
    float c[APART ? 2 : 1][8], s[APART ? 2 : 1][8];  // not APART: 8 pairs (kPairsHalf), or 4 of each slot (kPairsNext)
    if (pos >= 0) {
        const float *cp = a.rope.cos + (int64_t)pos * half, *sp = a.rope.sin + (int64_t)pos * half;
        if constexpr (APART) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = D / 2 * x + 8 * r;
                if (i >= 2 * half) continue;
                load8f(cp + (i < half ? i : i - half), c[x]);
                load8f(sp + (i < half ? i : i - half), s[x]);
            }
        } else if (style == kPairsHalf) {
            load8f(cp + 8 * r, c[0]);
            load8f(sp + 8 * r, s[0]);
        } else if (style == kPairsNext) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = D / 2 * x + 8 * r;
                if (i >= 2 * half) continue;
                const float4 u = __ldg(reinterpret_cast<const float4*>(cp + i / 2)), v = __ldg(reinterpret_cast<const float4*>(sp + i / 2));
                c[0][4 * x] = u.x, c[0][4 * x + 1] = u.y, c[0][4 * x + 2] = u.z, c[0][4 * x + 3] = u.w;
                s[0][4 * x] = v.x, s[0][4 * x + 1] = v.y, s[0][4 * x + 2] = v.z, s[0][4 * x + 3] = v.w;
            }
        }
        if constexpr (APPEND) {
            page = pos / a.pt.page_size;
            in_page = pos - page * a.pt.page_size;
        }
    }
    for (int g = g0; g < g1; ++g) {
        float x[2][8];
        const bool live = g * ROWS + sub < heads;
        int kind, h;
        place(g, kind, h);
        asm volatile("cp.async.wait_group %0;" ::"n"(R::STAGES - 1) : "memory");
        {
            const uint8_t* at = mine + (g - g0) % R::STAGES * (R::UNITS * 512);
            load8(at, 0, T{}, x[0]);
            load8(at, 1, T{}, x[1]);
        }
        fetch(g + R::STAGES);
        const float* w = kind == 0 ? a.rope.q_weight : kind == 1 ? a.rope.k_weight : nullptr;
        if (__any_sync(0xffffffffu, live && w)) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = __fadd_rn(__fmul_rn(x[0][j], x[0][j]), __fmul_rn(x[1][j], x[1][j]));
            const float mean = __fmul_rn(group_tree<D>(p, lane), 1.0f / D);  // D is a power of two: the quotient
            const float n = __frcp_rn(__fsqrt_rn(__fadd_rn(mean, a.rope.eps)));
            if (live && w) {
                float wv[8];
                const float2 n2 = make_float2(n, n);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    load8f(w + D / 2 * y + 8 * r, wv);
#pragma unroll
                    for (int j = 0; j < 8; j += 2) put(x[y], j, mul2(mul2(pair(x[y], j), n2), pair(wv, j)));
                }
            }
        }
        if constexpr (APART) {  // partners are whole chunks of 8, in another lane or slot
            float z[2][8];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int i = D / 2 * y + 8 * r, chunk = (i < half ? i + half : i - half) / 8;
                const bool turn = i < 2 * half;
                const int from = sub * LPR + (turn ? chunk % LPR : r);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v0 = __shfl_sync(0xffffffffu, x[0][j], from), v1 = __shfl_sync(0xffffffffu, x[1][j], from);
                    const float own = __fmul_rn(x[y][j], c[y][j]), other = __fmul_rn(chunk < LPR ? v0 : v1, s[y][j]);
                    z[y][j] = !turn || kind == 2 ? x[y][j] : i < half ? __fsub_rn(own, other) : __fadd_rn(own, other);
                }
            }
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[y][j] = z[y][j];
        } else if (style == kPairsHalf) {
            if (kind != 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u = x[0][j], v = x[1][j];
                    x[0][j] = __fsub_rn(__fmul_rn(u, c[0][j]), __fmul_rn(v, s[0][j]));
                    x[1][j] = __fadd_rn(__fmul_rn(v, c[0][j]), __fmul_rn(u, s[0][j]));
                }
            }
        } else if (style == kPairsNext) {
#pragma unroll
            for (int y = 0; y < 2; ++y)
                if (kind != 2 && D / 2 * y + 8 * r < 2 * half) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float u = x[y][2 * j], v = x[y][2 * j + 1], cc = c[0][4 * y + j], ss = s[0][4 * y + j];
                        x[y][2 * j] = __fsub_rn(__fmul_rn(u, cc), __fmul_rn(v, ss));
                        x[y][2 * j + 1] = __fadd_rn(__fmul_rn(v, cc), __fmul_rn(u, ss));
                    }
                }
        }
        if (pos < 0) {  // padding
#pragma unroll
            for (int j = 0; j < 8; ++j) x[0][j] = x[1][j] = 0.0f;
        }
        O* out = reinterpret_cast<O*>(kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out);
        if (out) out += (t * (kind == 0 ? a.n_heads : a.n_kv_heads) + h) * D + 8 * r;
        const bool encode = APPEND && live && kind != 0;
        if (live && !encode) {
            store8(out, x[0]);
            store8(out + D / 2, x[1]);
        }
        if constexpr (APPEND) {
            if (!__any_sync(0xffffffffu, encode)) continue;
            int64_t row = -1;
            if (encode && pos >= 0) {
                const int pg = __ldg(a.pt.pages + ((int64_t)seq * a.n_kv_heads + h) * a.pt.max_pages + page);
                if (pg >= 0 && pg < a.pt.n_pages)
                    row = (int64_t)pg * a.pt.page_size + in_page;
                else if (r == 0)
                    raise_device_error(a.err, BC_DEVERR_PAGE);
            }
            // sign bytes, mean |z|, residual, codes: encode_row's arithmetic.  |z - rec| is ||z| - s|
            // and the code of z that of |z| with z's sign (rounding is symmetric), `pos_mask` the reference's
            // z >= 0 (so -0 is, NaN is not).
            float p[8];
            uint32_t byte[2] = {0, 0}, pos_mask[2][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = __fadd_rn(fabsf(x[0][j]), fabsf(x[1][j]));
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    asm("set.ge.u32.f32 %0, %1, 0f00000000;" : "=r"(pos_mask[y][j]) : "f"(x[y][j]));
                    byte[y] |= pos_mask[y][j] & (1u << j);
                }
            }
            const float mean = __fmul_rn(group_tree<D>(p, lane), 1.0f / D);
            const uint16_t sb = f2h_bits(mean);
            const float held = __half2float(__ushort_as_half(sb));
            const float scale = res == BC_RES_FP16_SCALE ? held : mean;
            uint32_t word[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                uint32_t v = byte[y] << (8 * (r & 3));
                v |= __shfl_xor_sync(0xffffffffu, v, 1);
                word[y] = v | __shfl_xor_sync(0xffffffffu, v, 2);
            }
            const bc_kv_planes& P = kind == 1 ? a.K : a.V;
            if (row >= 0) {
                uint32_t* sg = reinterpret_cast<uint32_t*>(P.sign) + row * (D / 32);
                if ((r & 3) < 2) sg[(r & 1) * (D / 64) + r / 4] = word[r & 1];
                if (r == 0) reinterpret_cast<uint16_t*>(P.bscale)[row] = sb;
            }
            // |residual * inv| <= 7 (1 + 2^-23), so adding 1.5 * 2^23 + 8 rounds to the nearest whole number,
            // ties to even, and leaves code + 8 in the low bits
            constexpr float kRound = 12582920.0f;
            float rs = 0.0f;
            bool any = false;
            if (res != BC_RES_NONE) {
                float most = 0.0f;
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        // the residual as if z were positive, then its code as fp32 bits
                        x[y][j] = __fsub_rn(fabsf(x[y][j]), scale);
                        most = fmaxf(most, fabsf(x[y][j]));
                    }
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                float inv = most > 0.0f ? __fdiv_rn(7.0f, most) : 0.0f;
                if (inv == INFINITY) {  // most below 2^-125: the clamped products are +-7 and 0 (and both scales 0)
                    inv = 1.0f;
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[y][j] = x[y][j] != 0.0f ? copysignf(7.0f, x[y][j]) : 0.0f;
                }
                any = inv > 0.0f;  // else (rows of zeros, rows that are not finite) all codes are 0
                const uint16_t rb = f2h_bits(most);
                rs = __half2float(__ushort_as_half(rb));
                uint32_t nib[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    uint32_t q[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t m = __float_as_uint(__fmul_rn(x[y][j], inv)) ^ (~pos_mask[y][j] & 0x80000000u);
                        x[y][j] = __fadd_rn(__uint_as_float(m), kRound);
                        q[j] = __float_as_uint(x[y][j]);
                    }
                    // nibble byte t (of 4) holds bits t (low) and t + 4 (high) of the sign byte
                    const uint32_t lo = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                    const uint32_t hi = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
                    nib[y] = any ? (lo & 0x0F0F0F0Fu) | (hi << 4 & 0xF0F0F0F0u) : 0x88888888u;
                    nib[y] = transpose4(nib[y], r & 3);  // nibble word of t = r % 4, sign bytes 4 (r / 4) .. + 3
                }
                if (row >= 0) {
                    const int t4 = r & 3, g4 = r / 4;
                    uint8_t* nb = reinterpret_cast<uint8_t*>(P.nib);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int chunk = D == 128 ? t4 : D == 256 ? 4 * y + t4 : t4 / 2;
                        const int at = D == 128 ? 8 * y + 4 * g4 : D == 256 ? 4 * g4 : 8 * (t4 & 1) + 4 * y;
                        *reinterpret_cast<uint32_t*>(nb + nib_chunk_offset(row, chunk, D) + at) = nib[y];
                    }
                    if (r == 0) reinterpret_cast<uint16_t*>(P.rscale)[row] = rb;
                }
            }
            if (encode && out) {  // the rows as the planes hold them
                // codes of 0 times an infinite scale are NaN here too
                const uint32_t base = __float_as_uint(any || rs == 0.0f ? held : NAN);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[j] = __uint_as_float(base ^ (~pos_mask[y][j] & 0x80000000u));
                        if (any) {
                            // code / 7 rounded to nearest: one correction of the product with 1 / 7 (Markstein's)
                            constexpr float k7 = 1.0f / 7.0f;
                            const float code = __fsub_rn(x[y][j], kRound), q0 = __fmul_rn(code, k7);
                            const float q = __fmaf_rn(__fmaf_rn(q0, -7.0f, code), k7, q0);
                            v[j] = __fadd_rn(v[j], __fmul_rn(q, rs));
                        }
                        if (row < 0) v[j] = 0.0f;
                    }
                    store8(out + D / 2 * y, v);
                }
            }
        }
    }
}

// Whether k_rope_lanes takes a call, and in which of its styles.
static bool lanes_style(const RopeArgs& a, int head_dim, uintptr_t size, bool append, int* style) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return false;
    const bc_heads* in[3] = {&a.q, &a.k, &a.v};
    const int n[3] = {a.n_heads, a.n_kv_heads, append ? a.n_kv_heads : 0};
    for (int i = 0; i < 3; ++i)
        if (n[i] && (!bc_aligned(in[i]->data, 16) || in[i]->token_stride * (int64_t)size % 16 ||
                     in[i]->head_stride * (int64_t)size % 16))
            return false;
    const void* p[7] = {a.q_out, a.k_out, a.v_out, a.rope.q_weight, a.rope.k_weight, a.rope.cos, a.rope.sin};
    for (const void* x : p)
        if (!bc_aligned(x, 16)) return false;
    const int rot = a.rope.rotary_dim;
    *style = kPairsNone;
    if (!a.rope.cos) return true;
    if (a.rope.interleaved) {
        *style = kPairsNext;
        return rot % 8 == 0;
    }
    *style = rot == head_dim ? kPairsHalf : kPairsApart;
    return rot % 16 == 0;
}

template <int D, typename T, typename O, bool APPEND>
static int launch_lanes(const RopeArgs& a, int style, int res, cudaStream_t st) {
    const int heads = a.n_heads + (APPEND ? 2 : 1) * a.n_kv_heads;
    const int groups = (heads + Lanes<D>::ROWS - 1) / Lanes<D>::ROWS;
    // runs of heads: long ones keep a token's cosines, short ones fill the GPU (some 32 warps on each of 148 SMs)
    const int64_t fill = a.n_tokens * groups / (148 * 32);
    const int per = (int)(fill < 1 ? 1 : fill > groups ? groups : fill);
    const int64_t blocks = (a.n_tokens * ((groups + per - 1) / per) + kRopeWarps - 1) / kRopeWarps;
    if (blocks > INT32_MAX) return BC_ERR_TOO_LARGE;
    if (style == kPairsApart)
        k_rope_lanes<D, T, O, APPEND, true><<<(unsigned)blocks, kRopeWarps * 32, 0, st>>>(a, style, per, res);
    else
        k_rope_lanes<D, T, O, APPEND, false><<<(unsigned)blocks, kRopeWarps * 32, 0, st>>>(a, style, per, res);
    BC_LAUNCH_CHECK();
    return BC_OK;
}

template <typename T, typename O, bool APPEND, int RES>
static int launch_rope(const RopeArgs& a, int head_dim, cudaStream_t st) {
    int style = 0;
    if (lanes_style(a, head_dim, sizeof(T), APPEND, &style)) {
        if (head_dim == 64) return launch_lanes<64, T, O, APPEND>(a, style, RES, st);
        if (head_dim == 128) return launch_lanes<128, T, O, APPEND>(a, style, RES, st);
        return launch_lanes<256, T, O, APPEND>(a, style, RES, st);
    }
    const int64_t jobs = a.n_tokens * (a.n_heads + (APPEND ? 2 : 1) * (int64_t)a.n_kv_heads);
    const int64_t blocks = (jobs + kRopeWarps - 1) / kRopeWarps;
    if (blocks > INT32_MAX) return BC_ERR_TOO_LARGE;
    switch (head_dim / 32) {
#define BC_ROPE_CASE(N) \
    case N: k_rope_rows<N, T, O, APPEND, RES><<<(unsigned)blocks, kRopeWarps * 32, 0, st>>>(a); break;
        BC_ROPE_CASE(1)
        BC_ROPE_CASE(2)
        BC_ROPE_CASE(3)
        BC_ROPE_CASE(4)
        BC_ROPE_CASE(5)
        BC_ROPE_CASE(6)
        BC_ROPE_CASE(7)
        BC_ROPE_CASE(8)
#undef BC_ROPE_CASE
        default: return BC_ERR_HEAD_DIM;
    }
    BC_LAUNCH_CHECK();
    return BC_OK;
}

template <typename T>
static int rope_out(const RopeArgs& a, int head_dim, int out_dtype, cudaStream_t st) {
    switch (out_dtype) {
        case BC_DTYPE_F16: return launch_rope<T, __half, false, BC_RES_NONE>(a, head_dim, st);
        case BC_DTYPE_BF16: return launch_rope<T, __nv_bfloat16, false, BC_RES_NONE>(a, head_dim, st);
        default: return launch_rope<T, float, false, BC_RES_NONE>(a, head_dim, st);
    }
}

template <typename T>
static int append_res(const RopeArgs& a, int head_dim, int residual_mode, cudaStream_t st) {
    switch (residual_mode) {
        case BC_RES_NONE: return launch_rope<T, __half, true, BC_RES_NONE>(a, head_dim, st);
        case BC_RES_FP16_SCALE: return launch_rope<T, __half, true, BC_RES_FP16_SCALE>(a, head_dim, st);
        default: return launch_rope<T, __half, true, BC_RES_FP32_SCALE>(a, head_dim, st);
    }
}

static bool valid_dtype(int t) { return t == BC_DTYPE_F16 || t == BC_DTYPE_BF16 || t == BC_DTYPE_F32; }
static uintptr_t dtype_size(int t) { return t == BC_DTYPE_F32 ? 4 : 2; }

static int check_rope(const bc_rope& r, int head_dim) {
    if ((r.cos == nullptr) != (r.sin == nullptr)) return BC_ERR_ARG;
    if (r.cos && (r.rotary_dim < 2 || r.rotary_dim > head_dim || r.rotary_dim % 2 != 0 || r.n_positions <= 0))
        return BC_ERR_ARG;
    if ((r.q_weight || r.k_weight) && !(r.eps >= 0.0f)) return BC_ERR_ARG;
    const void* p[4] = {r.cos, r.sin, r.q_weight, r.k_weight};
    for (const void* x : p)
        if (!bc_aligned(x, 4)) return BC_ERR_ALIGN;
    return BC_OK;
}

static int check_heads(const bc_heads& x, int n, int dtype) {
    if (n == 0) return BC_OK;
    if (!x.data) return BC_ERR_ARG;
    return bc_aligned(x.data, dtype_size(dtype)) ? BC_OK : BC_ERR_ALIGN;
}

}  // namespace bc

using namespace bc;

extern "C" {

int bc_qk_norm_rope(bc_heads q, bc_heads k, const int32_t* positions, bc_rope rope, void* q_out, void* k_out,
                    int64_t n_tokens, int n_heads, int n_kv_heads, int head_dim, int dtype, int out_dtype,
                    void* stream) {
    if (!bc_valid_head_dim(head_dim)) return BC_ERR_HEAD_DIM;
    if (n_tokens < 0 || n_heads < 0 || n_kv_heads < 0 || !valid_dtype(dtype) || !valid_dtype(out_dtype))
        return BC_ERR_ARG;
    int rc = check_rope(rope, head_dim);
    if (rc) return rc;
    if (n_tokens == 0 || n_heads + (int64_t)n_kv_heads == 0) return BC_OK;
    if (!positions || (n_heads && !q_out) || (n_kv_heads && !k_out)) return BC_ERR_ARG;
    if ((rc = check_heads(q, n_heads, dtype)) || (rc = check_heads(k, n_kv_heads, dtype))) return rc;
    if (!bc_aligned(positions, 4) || !bc_aligned(q_out, dtype_size(out_dtype)) ||
        !bc_aligned(k_out, dtype_size(out_dtype)))
        return BC_ERR_ALIGN;
    RopeArgs a{};
    a.q = q;
    a.k = k;
    a.positions = positions;
    a.rope = rope;
    a.q_out = q_out;
    a.k_out = k_out;
    a.n_tokens = n_tokens;
    a.n_heads = n_heads;
    a.n_kv_heads = n_kv_heads;
    a.err = bc_device_error_ptr();
    if (!a.err) return BC_ERR_CUDA_BASE;
    cudaStream_t st = (cudaStream_t)stream;
    switch (dtype) {
        case BC_DTYPE_F16: return rope_out<__half>(a, head_dim, out_dtype, st);
        case BC_DTYPE_BF16: return rope_out<__nv_bfloat16>(a, head_dim, out_dtype, st);
        default: return rope_out<float>(a, head_dim, out_dtype, st);
    }
}

int bc_append_qkv_paged(bc_heads q, bc_heads k, bc_heads v, const int32_t* seq_ids, const int32_t* positions,
                        bc_rope rope, void* q_out, bc_kv_planes K, bc_kv_planes V, bc_page_table pt, void* k_hat,
                        void* v_hat, int64_t n_tokens, int n_seqs, int n_heads, int n_kv_heads, int head_dim,
                        int dtype, int residual_mode, void* stream) {
    if (!bc_valid_head_dim(head_dim)) return BC_ERR_HEAD_DIM;
    if (n_tokens < 0 || n_seqs < 0 || n_heads < 0 || n_kv_heads <= 0 || !valid_dtype(dtype)) return BC_ERR_ARG;
    if (residual_mode < BC_RES_NONE || residual_mode > BC_RES_FP32_SCALE) return BC_ERR_ARG;
    int rc = check_rope(rope, head_dim);
    if (rc) return rc;
    if (n_tokens == 0) return BC_OK;
    if (!pt.pages || pt.page_size <= 0 || pt.page_size % 128 != 0 || pt.n_pages <= 0 || pt.max_pages <= 0)
        return BC_ERR_ARG;
    if (!positions || !seq_ids || (n_heads && !q_out) || (k_hat == nullptr) != (v_hat == nullptr)) return BC_ERR_ARG;
    if ((rc = check_heads(q, n_heads, dtype)) || (rc = check_heads(k, n_kv_heads, dtype)) ||
        (rc = check_heads(v, n_kv_heads, dtype)))
        return rc;
    const bool res = residual_mode != BC_RES_NONE;
    const void* planes[8] = {K.sign, K.bscale, V.sign, V.bscale, K.nib, K.rscale, V.nib, V.rscale};
    for (int i = 0; i < (res ? 8 : 4); ++i) {
        if (!planes[i]) return BC_ERR_ARG;
        if (!bc_aligned(planes[i], 16)) return BC_ERR_ALIGN;
    }
    if (!bc_aligned(positions, 4) || !bc_aligned(seq_ids, 4) || !bc_aligned(pt.pages, 4) || !bc_aligned(q_out, 2) ||
        !bc_aligned(k_hat, 2) || !bc_aligned(v_hat, 2))
        return BC_ERR_ALIGN;
    RopeArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.positions = positions;
    a.seq_ids = seq_ids;
    a.rope = rope;
    a.q_out = q_out;
    a.k_out = k_hat;
    a.v_out = v_hat;
    a.K = K;
    a.V = V;
    a.pt = pt;
    a.n_tokens = n_tokens;
    a.n_seqs = n_seqs;
    a.n_heads = n_heads;
    a.n_kv_heads = n_kv_heads;
    a.err = bc_device_error_ptr();
    if (!a.err) return BC_ERR_CUDA_BASE;
    cudaStream_t st = (cudaStream_t)stream;
    switch (dtype) {
        case BC_DTYPE_F16: return append_res<__half>(a, head_dim, residual_mode, st);
        case BC_DTYPE_BF16: return append_res<__nv_bfloat16>(a, head_dim, residual_mode, st);
        default: return append_res<float>(a, head_dim, residual_mode, st);
    }
}

}  // extern "C"
