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

template <typename T, typename O, bool APPEND, int RES>
static int launch_rope(const RopeArgs& a, int head_dim, cudaStream_t st) {
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
