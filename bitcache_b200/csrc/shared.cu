// Decode attention of a batch over a paged cache whose sequences share
// prefixes: positions [0, prefix) of a group of sequences are read once for all
// of the group's query heads, the rest once per sequence.  Ragged lengths, held
// in device memory.  sm_100a.
//
// Mathematics (as bc_decode_attention), query row q, key with sign bits k, codes
// n and scales bs, rs, value likewise:
//   s   = (bs mean|q| (sgn q . sgn k) + rs / 7 (q . n)) / sqrt(d)
//   out = sum_s softmax(s) (bs_v sgn v + rs_v / 7 n_v)
// Work is a flat list: an item is one block of up to 8 query rows of one kv head
// against a prefix of a group or the rest of a sequence, in tiles of 32 keys.
// The warps of the grid divide the list evenly, each item weighing its tiles and
// a constant for its start and end, so ragged lengths need no plan on the host.
// A warp's stretch of an item is a piece, whose record (U, l, o) k_shared_merge
// joins with the row's other pieces.  A warp works alone: its own ring of tiles
// (cp.async), its own softmax state, no barrier but the one after the list's
// sums.  (With the four warps of a CTA on the 32-key quarters of one tile, the
// merge and the barriers at every piece cost more than the products of a short
// sequence: 51 of 84 us busy at 16 sequences of 8192 shared and 64 own keys.)
//
// Rows are the narrow side of every product (mma.sync m16n8k16, fp16 in, fp32
// accumulators): the 16 rows of A are keys in the scores and dims in the values,
// the 8 columns of B are query rows.  A is built in registers from the packed
// bytes: masked in place, a sign bit or nibble is an fp16 subnormal, 2^(p - 24)
// times its value at bit position p.  For the scores that is A already (the
// powers of two go into the query's side, the offset 8 of the codes and the 0/1
// of the sign bits into a constant per row); for the values one fma makes it the
// signed number times 2^-10, so that the long sums stay centred: the tensor
// cores cut what they add to, and with the offset left in, a sum over 200000
// keys lost 3%.  A key's scales multiply its few scores, and its probabilities
// before they become the value product's B operand: P1 = e bs, P2 = e rs / 7,
// rounded to fp16.  They keep at least 11 significant bits down to 2^-22 of a
// row's largest one: e is 2^(s - U) with U such that the largest P lies between
// 2^8 and 2^15.
//
// What bounds it is a tile's chain (copies, scores, weights, values) in each warp
// and the instructions of building A, not HBM: 128 sequences of 16 prompts up to 4000
// keys, 16 heads of 64, take 45 us (77 MB: 1.7 TB/s), 48 ragged sequences up to 6000
// keys, sign bits only, 8 heads of 256, 55 us (75 MB: 1.4 TB/s).
#include "shared.cuh"
#include "shared_tc.h"

namespace bc {
namespace {

constexpr int kShWarps = kShThreads / 32;
constexpr int kShTile = 32;        // keys per tile
static_assert(kShTile == 1 << 5, "the list's shift");
constexpr int kShRows = 8;         // query rows per item
constexpr int kShStages = 2;
constexpr int kShItemCost = 2;     // an item's start and end, in tiles
constexpr int kShMaxWorkers = 148 * 16;  // bound of the workers, for the workspace's size
constexpr int kShTcWorkers = 148;        // CTAs of the prefix kernel, one per SM

template <int D, bool COMP>
struct ShCfg {
    static constexpr int NW = D / 32;
    static constexpr int SIGN_B = kShTile * D / 8;
    static constexpr int NIB_B = COMP ? kShTile * D / 2 : 0;
    static constexpr int SC_B = kShTile * 2;
    static constexpr int HALF_B = SIGN_B + NIB_B + SC_B * (COMP ? 2 : 1);  // K (or V) part of a stage
    static constexpr int NIB_OFF = SIGN_B;
    static constexpr int BS_OFF = SIGN_B + NIB_B;
    static constexpr int RS_OFF = BS_OFF + SC_B;
    static constexpr int Q_ROW = 2 * D + 16;  // padded: the rows' 2-byte reads spread over the banks
    static constexpr int Q_OFF = 2 * HALF_B;  // the query rows, with the first tile of an item
    static constexpr int STAGE_B = Q_OFF + kShRows * Q_ROW;
    static constexpr int WARP_B = kShStages * STAGE_B;
    static constexpr int SCAN_OFF = kShWarps * WARP_B;
    static constexpr int SMEM_B = SCAN_OFF + (kShThreads + 1) * 8 + 8;
};

// ---- fragments -------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void sh_ldsm4(const uint8_t* row, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(row)) : "memory");
}
// Two 16x16 byte matrices, transposed: lanes 0-15 / 16-31 give the rows of the
// first / second; lane (g, q) gets bytes g and g + 8 of rows 4q .. 4q + 3.
__device__ __forceinline__ void sh_ldsm_t2(const uint8_t* row, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(row)) : "memory");
}
__device__ __forceinline__ void sh_ldsm_t1(const uint8_t* row, uint32_t& r0, uint32_t& r1) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x1.trans.shared.b8 {%0,%1}, [%2];"
                 : "=r"(r0), "=r"(r1)
                 : "r"(smem_u32(row)) : "memory");
}
__device__ __forceinline__ void sh_cp16(uint8_t* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// fp16 pairs.  2^e, e in [-14, 15], in both halves:
__device__ constexpr uint32_t pow2_h2(int e) { return (uint32_t)(e + 15) * 0x04000400u; }
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Value operands carry the factor 2^-10 (kShValue undoes it).
constexpr float kShValue = 1024.0f;
// Bits t and t + 16 of w (t <= 9) as +-2^-10: b 2^(t - 24) -> b 2^-9 - 2^-10.
__device__ __forceinline__ uint32_t sign_h2(uint32_t w, int t) {
    return fma_h2(w & (0x00010001u << t), pow2_h2(15 - t), 0x8000'8000u | pow2_h2(-10));
}
// Nibbles at bits 0-3 and 16-19 (hi: 4-7 and 20-23) of w, code + 8, as code 2^-10.
__device__ __forceinline__ uint32_t code_h2(uint32_t w, int hi) {
    return fma_h2(w & (hi ? 0x00F000F0u : 0x000F000Fu), pow2_h2(hi ? 10 : 14), 0x8000'8000u | pow2_h2(-7));
}

// The query rows as B operands, and what the scores need of each row.
// A pair of sign bits at position p is worth 2^(p - 24): its +-1 is +-2^(9 - p)
// here, the product's unit 2^-15.  A nibble at bits 0-3 / 4-7 is worth 2^-24 /
// 2^-20: its q is 16 q / q times a power of two u that puts the row's largest
// element at 2^10 .. 2^11, the product's unit 2^-20 / u.
template <int D, bool COMP>
struct ShQuery {
    uint32_t sign[D / 16][2];
    uint32_t code[COMP ? D / 16 : 1][2];
    float bco[2], boff[2], rco[2], roff[2];  // rows 2q, 2q + 1: score = bs (bco D1 - boff) + rs (rco D2 - roff)
};

// Dim of element `half` (0, 1) of register r of k step s in the sign part / code part, lane column q.
template <int D>
__device__ __forceinline__ int sign_dim(int s, int r, int half, int q) {
    const int p = 2 * s + r;  // pair within the lane's D / 8
    if constexpr (D >= 128) return 32 * (q + 4 * (p / 16)) + p % 16 + 16 * half;
    if constexpr (D == 64) return 32 * (q / 2) + 8 * (q % 2) + p + 16 * half;
    return 4 * q + p + 16 * half;  // D == 32
}
// Where pair p (of 16 in a word) is masked: in place, or 6 lower in the word shifted by 6.
__device__ constexpr int sign_pos(int p) { return p % 16 < 10 ? p % 16 : p % 16 - 6; }
template <int D>
__device__ __forceinline__ int code_dim(int s, int r, int half, int q) {
    const int c = s / 2, n = 2 * (s % 2) + r + 4 * half;  // chunk, nibble of its word q
    return nib_dim(D, c, 4 * q + n / 2, n % 2);
}

template <int D, bool COMP>
__device__ __forceinline__ void sh_load_query(const SharedArgs& a, const ShList& L, const ShCursor& c,
                                              const uint8_t* qrows, ShQuery<D, COMP>& Q) {
    using C = ShCfg<D, COMP>;
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
    const bool live = sh_query(a, L, c, c.blk * kShRows + g8, D) != nullptr;
    const __half* row = reinterpret_cast<const __half*>(qrows + g8 * C::Q_ROW);
    float sum = 0.0f, mag = 0.0f, top = 0.0f, sgn = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float f0 = live ? __half2float(row[sign_dim<D>(s, r, 0, q)]) : 0.0f;
            const float f1 = live ? __half2float(row[sign_dim<D>(s, r, 1, q)]) : 0.0f;
            Q.sign[s][r] = pow2_h2(9 - sign_pos(2 * s + r)) | (f0 >= 0.0f ? 0u : 0x8000u) | (f1 >= 0.0f ? 0u : 0x80000000u);
            mag += fabsf(f0) + fabsf(f1);
            sum += f0 + f1;
            sgn += (f0 >= 0.0f ? 1.0f : -1.0f) + (f1 >= 0.0f ? 1.0f : -1.0f);
            top = fmaxf(top, fmaxf(fabsf(f0), fabsf(f1)));
        }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        mag += __shfl_xor_sync(0xffffffffu, mag, o);
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        sgn += __shfl_xor_sync(0xffffffffu, sgn, o);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    // u: the largest element to 2^10 .. 2^11 (a row of zeros, or with an infinity: 1)
    const int ex = (__float_as_int(top) >> 23) - 127;
    const float u = top > 0.0f && ex < 16 ? exp2i(10 - ex) : 1.0f;
    if constexpr (COMP) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float w = r == 0 ? 16.0f * u : u;  // r = 0: nibbles 0-3 and 16-19 of the word, or of it shifted by 8
                const float f0 = live ? __half2float(row[code_dim<D>(s, r, 0, q)]) : 0.0f;
                const float f1 = live ? __half2float(row[code_dim<D>(s, r, 1, q)]) : 0.0f;
                Q.code[s][r] = pack_h2(f0 * w, f1 * w);
            }
    }
    const float scale = kShLog2e * rsqrtf((float)D);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int from = 4 * (2 * q + j);
        const float m = __shfl_sync(0xffffffffu, mag, from) * (1.0f / D) * scale;
        const float t = __shfl_sync(0xffffffffu, sum, from) * scale * (8.0f / 7.0f);
        const float w = __shfl_sync(0xffffffffu, u, from);
        Q.bco[j] = m * 65536.0f;  // sgn q . sgn k = 2 sum(sgn q bit) - sum(sgn q), in units of 2^-15
        Q.boff[j] = m * __shfl_sync(0xffffffffu, sgn, from);
        Q.rco[j] = scale * (1.0f / 7.0f) * 1048576.0f / w;
        Q.roff[j] = t;
    }
}

// Accumulators of one warp: o[mt][4] with rows of m-tile mt = 2c + h the dims
// nib_dim(D, c, g8 (+ 8), h), columns the query rows 2q, 2q + 1.
template <int D>
struct ShState {
    float o[D / 16][4];
    float U[2], l[2];  // per row 2q, 2q + 1: unit, and the sum of e over this lane's keys
};
template <int D>
__device__ __forceinline__ void sh_clear(ShState<D>& st) {
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[m][i] = 0.0f;
    st.U[0] = st.U[1] = kShNone;
    st.l[0] = st.l[1] = 0.0f;
}

// Position of matrix row r (0 .. 15) of a transposing load among its 16 keys:
// bytes 0, 2 of a lane's register are the k elements 2q, 2q + 1 and bytes 1, 3
// the elements 2q + 8, 2q + 9.
__device__ __forceinline__ int sh_key_of_row(int r) { return 2 * (r >> 2) + ((r >> 1) & 1) + 8 * (r & 1); }

// The 32 keys of a tile at key position kpos.
template <int D, bool COMP>
__device__ __forceinline__ void sh_consume(const ShQuery<D, COMP>& Q, ShState<D>& st, const uint8_t* sb, int kpos,
                                           int lo, int hi, bool masked) {
    using C = ShCfg<D, COMP>;
    constexpr int NW = C::NW;
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
    const uint8_t *ks = sb, *vs = sb + C::HALF_B;
    float s[2][4];
    // ---- scores of two blocks of 16 keys
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int kb = 16 * b;
        float d1[4] = {0.f, 0.f, 0.f, 0.f}, d2[4] = {0.f, 0.f, 0.f, 0.f};
        {
            constexpr int PAIRS = D / 8;  // pairs of dims per lane
            uint32_t w[2][D >= 256 ? 2 : 1];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t* row = reinterpret_cast<const uint32_t*>(ks) + (kb + g8 + 8 * x) * NW;
                if constexpr (D >= 128) {
#pragma unroll
                    for (int i = 0; i < D / 128; ++i) w[x][i] = row[q + 4 * i];
                } else if constexpr (D == 64) {
                    w[x][0] = row[q >> 1] >> (8 * (q & 1));
                } else {
                    w[x][0] = row[0] >> (4 * q);
                }
            }
#pragma unroll
            for (int k = 0; k < PAIRS / 2; ++k) {
                const int i = 2 * k / 16, p = 2 * k % 16;  // pairs p, p + 1 of word i
                const uint32_t w0 = p < 10 ? w[0][i] : w[0][i] >> 6, w1 = p < 10 ? w[1][i] : w[1][i] >> 6;
                const uint32_t m0 = 0x00010001u << sign_pos(p), m1 = m0 << 1;
                mma_f16(d1, w0 & m0, w1 & m0, w0 & m1, w1 & m1, Q.sign[k][0], Q.sign[k][1]);
            }
        }
        if constexpr (COMP) {
            const uint8_t* nib = ks + C::NIB_OFF + (kb >> 3) * 4 * D;
            // word q of chunk c of key g8 (x = 0) and g8 + 8 (x = 1)
            uint32_t n[NW][2];
            if constexpr (NW >= 4) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int c4 = 0; c4 < NW / 4; ++c4) {
                        uint32_t r[4];
                        sh_ldsm4(nib + x * 4 * D + c4 * 512 + lane * 16, r);
#pragma unroll
                        for (int i = 0; i < 4; ++i) n[4 * c4 + i][x] = r[i];
                    }
            } else {
                uint32_t r[4];  // D = 64: both chunks of both blocks; D = 32: the chunk of both blocks, twice
                sh_ldsm4(nib + (lane * 16) % (8 * D), r);
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int c = 0; c < NW; ++c) n[c][x] = r[x * NW + c];
            }
#pragma unroll
            for (int c = 0; c < NW; ++c) {
                mma_f16(d2, n[c][0] & 0x000F000Fu, n[c][1] & 0x000F000Fu, n[c][0] & 0x00F000F0u, n[c][1] & 0x00F000F0u,
                        Q.code[2 * c][0], Q.code[2 * c][1]);
                const uint32_t y0 = n[c][0] >> 8, y1 = n[c][1] >> 8;
                mma_f16(d2, y0 & 0x000F000Fu, y1 & 0x000F000Fu, y0 & 0x00F000F0u, y1 & 0x00F000F0u,
                        Q.code[2 * c + 1][0], Q.code[2 * c + 1][1]);
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int key = kb + g8 + 8 * x;
            const float bs = __half2float(reinterpret_cast<const __half*>(ks + C::BS_OFF)[key]);
            const float rs = COMP ? __half2float(reinterpret_cast<const __half*>(ks + C::RS_OFF)[key]) : 0.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float v = bs * (Q.bco[j] * d1[2 * x + j] - Q.boff[j]);
                if constexpr (COMP) v += rs * (Q.rco[j] * d2[2 * x + j] - Q.roff[j]);
                s[b][2 * x + j] = v;
            }
        }
    }
    // ---- value scales, the keys' own masks, and the unit U of each row
    float vb[2][2], vr[2][2], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int key = 16 * b + g8 + 8 * x;
            vb[b][x] = __half2float(reinterpret_cast<const __half*>(vs + C::BS_OFF)[key]);
            vr[b][x] = COMP ? __half2float(reinterpret_cast<const __half*>(vs + C::RS_OFF)[key]) * (1.0f / 7.0f) : 0.0f;
            // 2^grow bounds the larger scale; a key whose scales are next to 0 does not pull U down by more than 2^40
            const float grow = (float)max(-40, (__float_as_int(fmaxf(vb[b][x], vr[b][x])) >> 23) - 126);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float& v = s[b][2 * x + j];
                if (masked && (kpos + key < lo || kpos + key >= hi)) v = -INFINITY;
                top[j] = fmaxf(top[j], v + grow);
            }
        }
    if (__any_sync(0xffffffffu, top[0] - st.U[0] > 15.0f || top[1] - st.U[1] > 15.0f)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float m = top[j];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float U = m - st.U[j] > 15.0f ? m - 8.0f : st.U[j];
            const float f = exp2f(st.U[j] - U);
            st.U[j] = U;
            st.l[j] *= f;
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
                st.o[mt][j] *= f;
                st.o[mt][2 + j] *= f;
            }
        }
    }
    // ---- probabilities as B operands, and the value sums
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        uint32_t p1[2], p2[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float c1[2], c2[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float v = s[b][2 * x + j];
                const float e = exp2f(v - st.U[j]);
                st.l[j] += e;
                const bool out = masked && v == -INFINITY;  // a masked row's scales may be anything
                c1[j] = out ? 0.0f : e * vb[b][x];
                c2[j] = out ? 0.0f : e * vr[b][x];
            }
            p1[x] = movmatrix(pack_h2(c1[0], c1[1]));
            if constexpr (COMP) p2[x] = movmatrix(pack_h2(c2[0], c2[1]));
        }
        const int kb = 16 * b;
        const int key = kb + sh_key_of_row(lane & 15);
        uint32_t sg[D >= 256 ? 4 : 2], wd[4];
        if constexpr (D == 128) {
            sh_ldsm_t1(vs + key * 16, sg[0], sg[1]);
        } else if constexpr (D == 256) {
            uint32_t r[4];
            sh_ldsm_t2(vs + key * 32 + (lane >> 4) * 16, r);
#pragma unroll
            for (int i = 0; i < 4; ++i) sg[i] = r[i];
        } else if constexpr (D == 64) {
            sg[0] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sg[0] |= (uint32_t)vs[(kb + sh_key_of_row(4 * q + i)) * 8 + g8] << (8 * i);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                wd[i] = reinterpret_cast<const uint32_t*>(vs)[kb + sh_key_of_row(4 * q + i)] >> (2 * g8);
        }
#pragma unroll
        for (int c = 0; c < NW; c += 2) {
            uint32_t r[4];
            if constexpr (COMP) {
                // the 16 bytes of chunk c (lanes 16-31: chunk c + 1) of each key
                const int cc = NW > 1 ? c + (lane >> 4) : 0;
                sh_ldsm_t2(vs + C::NIB_OFF + (key >> 3) * 4 * D + cc * 128 + (key & 7) * 16, r);
            }
#pragma unroll
            for (int cx = 0; cx < (NW > 1 ? 2 : 1); ++cx)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float(&o)[4] = st.o[2 * (c + cx) + h];
                    uint32_t a0, a1, a2, a3;
                    if constexpr (D >= 128) {
                        const int w = (c + cx) / 4, t = (c + cx) % 4 + 4 * h;
                        a0 = sign_h2(sg[2 * w], t);
                        a1 = sign_h2(sg[2 * w + 1], t);
                        a2 = sign_h2(sg[2 * w] >> 8, t);
                        a3 = sign_h2(sg[2 * w + 1] >> 8, t);
                    } else if constexpr (D == 64) {
                        const int t = 2 * (c + cx) + 4 * h;
                        a0 = sign_h2(sg[0], t);
                        a1 = sign_h2(sg[0], t + 1);
                        a2 = sign_h2(sg[0] >> 8, t);
                        a3 = sign_h2(sg[0] >> 8, t + 1);
                    } else {
                        a0 = sign_h2(__byte_perm(wd[0], wd[2], 0x5410), h);
                        a1 = sign_h2(__byte_perm(wd[0], wd[2], 0x7632), h);
                        a2 = sign_h2(__byte_perm(wd[1], wd[3], 0x5410), h);
                        a3 = sign_h2(__byte_perm(wd[1], wd[3], 0x7632), h);
                    }
                    mma_f16(o, a0, a1, a2, a3, p1[0], p1[1]);
                    if constexpr (COMP) {
                        const uint32_t x0 = r[2 * cx], x1 = r[2 * cx + 1];
                        mma_f16(o, code_h2(x0, h), code_h2(x1, h), code_h2(x0 >> 8, h), code_h2(x1 >> 8, h), p2[0], p2[1]);
                    }
                }
        }
    }
}

// The piece's record: rows of D + 4 floats, o (in the order of sh_code_dim) then (U, l).
template <int D>
__device__ __forceinline__ void sh_flush(const ShState<D>& st, float* m) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float l = st.l[j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        float* row = m + (2 * q + j) * (D + 4);
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // byte g8 + 8x of chunk mt / 2, its nibble mt % 2
                const int n = 2 * (g8 % 4) + mt % 2;
                row[8 * (4 * (mt / 2) + g8 / 4 + 2 * x) + 2 * (n % 4) + n / 4] = st.o[mt][2 * x + j] * kShValue;
            }
        if (g8 == 0) *reinterpret_cast<float2*>(row + D) = make_float2(st.U[j], l);
    }
}

template <int D, bool COMP>
__global__ void __launch_bounds__(kShThreads) k_shared_rows(const SharedArgs a, const ShList L, bool overlap) {
    using C = ShCfg<D, COMP>;
    extern __shared__ __align__(128) uint8_t smem[];
    int64_t* scan = reinterpret_cast<int64_t*>(smem + C::SCAN_OFF);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Behind the prefix kernel (which has waited for all that this one reads) the CTAs
    // start as SMs fall free; one more CTA waits for it on behalf of the launches to come.
    if (overlap && blockIdx.x == gridDim.x - 1) {
        sh_let_next();
        sh_wait_before();
        return;
    }
    if (!overlap) sh_wait_before();
    sh_let_next();
    const int64_t total = sh_scan(a, L, scan);
    if (blockIdx.x == 0) {  // lengths outside the block table are cut, and said so
        const int64_t cap = (int64_t)a.pt.max_pages * a.pt.page_size;
        for (int b = tid; b < a.n_seqs; b += kShThreads)
            if (a.seq_lens[b] < 0 || a.seq_lens[b] > cap) raise_device_error(a.err, BC_DEVERR_INDEX);
        if (a.prefix_lens)
            for (int g = tid; g < a.n_groups; g += kShThreads)
                if (a.prefix_lens[g] < 0 || a.prefix_lens[g] > cap) raise_device_error(a.err, BC_DEVERR_INDEX);
    }
    const int n_workers = sh_workers(L, total);
    const int worker = blockIdx.x * kShWarps + warp;
    if (worker >= n_workers) return;
    ShCursor cur;
    sh_seek(a, L, scan, n_workers, worker, cur);
    if (cur.left <= 0) return;  // the stretch ends within its first item's start

    uint8_t* ring = smem + warp * C::WARP_B;
    ShCursor ahead = cur;
    bool ahead_new = true;   // the query rows travel with the first tile of each piece
    unsigned present = 0;    // bit s: the page of stage s is in the pool
    int in_page = 0;         // position of `ahead` in its page
    int64_t row = -1;        // plane row of `ahead`; -1: page outside the pool
    const int32_t* page = nullptr;
    auto issue = [&](int s) {
        uint8_t* dst = ring + s * C::STAGE_B;
        if (ahead_new) {
            const int pos = (ahead.x.tile0 + ahead.tile) * kShTile;
            const int j = pos / a.pt.page_size;
            in_page = pos - j * a.pt.page_size;
            page = a.pt.pages + ((int64_t)sh_lead(a, L, ahead) * a.n_kv + ahead.h) * a.pt.max_pages + j;
        }
        if (ahead_new || in_page == a.pt.page_size) {
            if (!ahead_new) {
                ++page;
                in_page = 0;
            }
            const int pg = __ldg(page);
            row = pg >= 0 && pg < a.pt.n_pages ? (int64_t)pg * a.pt.page_size + in_page : -1;
            if (row < 0 && lane == 0) raise_device_error(a.err, BC_DEVERR_PAGE);
        }
        if (row >= 0) {
            present |= 1u << s;
            auto part = [&](const bc_kv_planes& P, uint8_t* d) {
#pragma unroll
                for (int i = lane * 16; i < C::SIGN_B; i += 512) sh_cp16(d + i, (const uint8_t*)P.sign + row * (D / 8) + i);
                if constexpr (COMP) {
#pragma unroll
                    for (int i = lane * 16; i < C::NIB_B; i += 512)
                        sh_cp16(d + C::NIB_OFF + i, (const uint8_t*)P.nib + row * (D / 2) + i);
                }
                constexpr int SC = C::SC_B / 16;
                if (lane < SC * (COMP ? 2 : 1)) {
                    const uint8_t* src = (const uint8_t*)(lane < SC ? P.bscale : P.rscale) + row * 2 + (lane % SC) * 16;
                    sh_cp16(d + C::BS_OFF + lane * 16, src);
                }
            };
            part(a.K, dst);
            part(a.V, dst + C::HALF_B);
            row += kShTile;
        } else {
            present &= ~(1u << s);
        }
        in_page += kShTile;
        if (ahead_new)
            for (int i = lane; i < kShRows * (D / 8); i += 32) {
                const int r = i / (D / 8), at = i % (D / 8) * 8;
                const __half* src = sh_query(a, L, ahead, ahead.blk * kShRows + r, D);
                if (!src) break;
                uint8_t* to = dst + C::Q_OFF + r * C::Q_ROW + 2 * at;
                if (a.q_aligned)
                    sh_cp16(to, src + at);
                else
                    for (int k = 0; k < 8; ++k) reinterpret_cast<__half*>(to)[k] = src[at + k];
            }
        ahead_new = sh_next(a, L, ahead);
    };
#pragma unroll
    for (int s = 0; s < kShStages; ++s) {
        if (ahead.left > 0) issue(s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    ShQuery<D, COMP> Q;
    ShState<D> st;
    bool begin = true;
    for (int s = 0; cur.left > 0; s = s + 1 == kShStages ? 0 : s + 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kShStages - 1) : "memory");
        __syncwarp();
        const uint8_t* sb = ring + s * C::STAGE_B;
        if (begin) {
            sh_load_query<D, COMP>(a, L, cur, sb + C::Q_OFF, Q);
            sh_clear(st);
        }
        const int kpos = (cur.x.tile0 + cur.tile) * kShTile;
        if (present >> s & 1)
            sh_consume<D, COMP>(Q, st, sb, kpos, cur.x.lo, cur.x.hi, kpos < cur.x.lo || kpos + kShTile > cur.x.hi);
        __syncwarp();
        if (ahead.left > 0) issue(s);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (sh_piece_ends(cur)) sh_flush<D>(st, sh_record(a, L, cur, worker, D));
        begin = sh_next(a, L, cur);
    }
}

// Joins a query row's pieces, those of its group's prefix (list P) and of its own
// keys (list O, which may hold both): WPR warps per row.  All that the lengths tell
// is worked out before the wait for the launches that write the records; behind it
// a row's records come in one L2 round trip as long as they are few.
// (Four CTAs of one row each fit an SM, so that up to kShSplitRows rows are one wave; seven of four rows each,
// where the registers suffice: 4096 rows 73.8 us for the whole call, 78.3 with six.)
template <int D, int WPR>
__global__ void __launch_bounds__(kShThreads, WPR == 1 && D <= 128 ? 7 : 4) k_shared_merge(const SharedArgs a, const ShList P, const ShList O, bool two) {
    constexpr int VEC = D / 32;  // consecutive floats of a lane
    constexpr int AT_ONCE = WPR == 1 || VEC > 4 ? 8 : 16;  // records in flight
    static_assert(WPR == 1 || WPR == kShWarps, "a warp or a CTA per row");
    __shared__ int64_t scan[2][kShThreads + 1];
    __shared__ float parts[WPR > 1 ? kShWarps : 1][D], marks[2][kShWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % WPR;
    // (unsigned: the heads of all sequences are below 2^31)
    const unsigned head = WPR == 1 ? blockIdx.x * kShWarps + warp : blockIdx.x, slot = head / (unsigned)a.group;
    const int b = (int)(slot / (unsigned)a.n_kv), h = (int)(slot - (unsigned)b * a.n_kv), g = (int)(head - slot * a.group);
    const bool live = b < a.n_seqs;
    sh_let_next();
    // the lengths are older than the launches before this one, the records are theirs
    int64_t total[2], first[2] = {0, 0}, size[2];
    int n_workers[2], tiles[2], c0[2] = {0, 0}, count[2] = {0, 0};
    const float* rec[2] = {nullptr, nullptr};
    total[1] = sh_scan(a, O, scan[1]);
    total[0] = two ? sh_scan(a, P, scan[0]) : total[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const ShList& L = i ? O : P;
        const int want = i ? O.n_pre + (live ? b : 0) : live ? b / a.per : 0;
        size[i] = (int64_t)L.rows * (D + 4) * L.copies;
        n_workers[i] = tiles[i] = 0;
        if (i == 0 && L.n_pre == 0) continue;
        // the weight before entry `want`: the run's start, and the run's entries before it, lane by lane
        const int n = L.n_pre + L.n_own, chunk = (n + kShThreads - 1) / kShThreads, run = want / chunk;
        int64_t sum = 0;
        for (int e = run * chunk + lane; e < want; e += 32) sum += sh_weight(a, L, sh_entry(a, L, e));
        if (chunk > 1) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        const ShEntry x = sh_entry(a, L, want);
        if (!live || x.tiles == 0 || (i == 0 && sh_len(a, b) < x.hi)) continue;  // (a shorter sequence takes no part in the prefix)
        tiles[i] = x.tiles;
        n_workers[i] = sh_workers(L, total[i]);
        const int r = i == 0 ? (b % a.per) * a.group + g : g;
        const int it = h * x.blocks + r / L.rows;
        first[i] = scan[two ? i : 1][run] + sum + (int64_t)it * sh_item_weight(L, x);
        c0[i] = sh_worker_of(total[i], n_workers[i], first[i]);
        count[i] = (sh_worker_of(total[i], n_workers[i], first[i] + sh_item_weight(L, x) - 1) - c0[i] + 1) * L.copies;
        rec[i] = L.records + (sh_first_item(L, a.n_kv, want) + it + c0[i]) * size[i] + (r % L.rows) * (D + 4);
    }
    // record q: the prefix's (a worker's copies one after the other), then the own keys'; null where a
    // worker's stretch holds no tile of the item
    const int all = count[0] + count[1], copies = P.copies;
    auto record = [&](int q) -> const float* {
        const bool own = q >= count[0];
        const int at = own ? q - count[0] : q, c = own ? at : at / copies;
        const ShList& L = own ? O : P;
        const int64_t from = own ? first[1] : first[0], sum = own ? total[1] : total[0], step = own ? size[1] : size[0] / copies;
        const int n = own ? n_workers[1] : n_workers[0], w = c + (own ? c0[1] : c0[0]), t = own ? tiles[1] : tiles[0];
        if (q >= all || sh_tile_at(L, sh_begin(sum, n, w) - from, t) >= sh_tile_at(L, sh_begin(sum, n, w + 1) - from, t)) return nullptr;
        return (own ? rec[1] : rec[0]) + at * step;
    };
    float M = kShNone, sum = 0.0f, o[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) o[k] = 0.0f;
    const float* from = record(WPR * lane + mine);
    sh_wait_before();
#pragma unroll 1
    for (int base = 0; base < all; from = record((base += 32 * WPR) + WPR * lane + mine)) {
        const float2 ul = from ? __ldcg(reinterpret_cast<const float2*>(from + D)) : make_float2(kShNone, 0.0f);
        unsigned todo = __ballot_sync(0xffffffffu, from != nullptr);
        bool scaled = false;
        float w = 0.0f;
        while (todo) {
            float v[AT_ONCE][VEC];
            int src[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                src[u] = todo ? __ffs(todo) - 1 : -1;
                todo &= todo - 1;
                const float* x = reinterpret_cast<const float*>(
                                     __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(from), src[u] & 31)) + VEC * lane;
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[u][k] = 0.0f;
                if (src[u] >= 0) {
                    if constexpr (VEC >= 4) {
#pragma unroll
                        for (int k = 0; k < VEC; k += 4)
                            *reinterpret_cast<float4*>(&v[u][k]) = __ldcg(reinterpret_cast<const float4*>(x + k));
                    } else {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) v[u][k] = __ldcg(x + k);
                    }
                }
            }
            if (!scaled) {  // with the records on their way
                float top = ul.x;
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                const float U = fmaxf(M, top), f = exp2f(M - U);
                w = from ? exp2f(ul.x - U) : 0.0f;
                float l = ul.y * w;
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
                M = U;
                sum = sum * f + l;
#pragma unroll
                for (int k = 0; k < VEC; ++k) o[k] *= f;
                scaled = true;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const float wt = __shfl_sync(0xffffffffu, w, src[u] & 31);
                if (src[u] >= 0) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) o[k] += v[u][k] * wt;
                }
            }
        }
    }
    // no keys: zeros
    if constexpr (WPR == 1) {
        const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
        if (live) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.out[(int64_t)head * D + sh_code_dim(D, VEC * lane + k)] = __float2half_rn(o[k] * inv);
        }
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) parts[warp][VEC * lane + k] = o[k];
        if (lane == 0) {
            marks[0][warp] = M;
            marks[1][warp] = sum;
        }
        __syncthreads();
        float f[WPR], U = kShNone, l = 0.0f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) U = fmaxf(U, marks[0][i]);
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            f[i] = exp2f(marks[0][i] - U);
            l += marks[1][i] * f[i];
        }
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        if (live) {
            for (int at = threadIdx.x; at < D; at += kShThreads) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < WPR; ++i) x += parts[i][at] * f[i];
                a.out[(int64_t)head * D + sh_code_dim(D, at)] = __float2half_rn(x * inv);
            }
        }
    }
}

template <int D, bool COMP>
int sh_workers_on_device(int* n_workers) {
    constexpr int smem = ShCfg<D, COMP>::SMEM_B;
    static int cached[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return BC_ERR_CUDA_BASE + (int)e;
    if (dev < 0 || dev >= 64) return BC_ERR_UNSUPPORTED;
    if (!cached[dev]) {
        int sms = 0, occ = 0;
        e = cudaFuncSetAttribute(k_shared_rows<D, COMP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess)
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, k_shared_rows<D, COMP>, kShThreads, smem);
        if (e != cudaSuccess) return BC_ERR_CUDA_BASE + (int)e;
        if (occ <= 0) return BC_ERR_UNSUPPORTED;
        cached[dev] = min(sms * occ * kShWarps, kShMaxWorkers);
    }
    *n_workers = cached[dev];
    return BC_OK;
}

// Up to this many query rows the merge gives each a CTA's four warps, which share its records, else a warp.
// One warp / four: 128 rows 16.1 / 12.2 us (the whole call), 256 rows 213 / 194, 512 rows 65.2 / 58.4; 768 rows
// 54.9 / 58.9, 4096 rows 74.2 / 105.8, where the CTAs' sums over the list cost more than the records.
constexpr int64_t kShSplitRows = 4 * 148;

// The prefix kernel takes the prefixes when `tc` is given, else the rows kernel has both.
template <int D, bool COMP>
int sh_run(const SharedArgs& a, ShList& L, const ShList* tc, void* scratch, cudaStream_t st) {
    int rc = sh_workers_on_device<D, COMP>(&L.n_workers);
    if (!rc && tc) rc = sh_tc_run(a, *tc, scratch, D, COMP, st);
    if (rc) return rc;
    const int64_t rows = (int64_t)a.n_seqs * a.n_kv * a.group;
    const ShList& P = tc ? *tc : L;
    cudaError_t e = sh_launch(k_shared_rows<D, COMP>, (L.n_workers + kShWarps - 1) / kShWarps + (tc ? 1 : 0), kShThreads,
                              ShCfg<D, COMP>::SMEM_B, st, a, L, tc != nullptr);
    if (e == cudaSuccess)
        e = rows <= kShSplitRows ? sh_launch(k_shared_merge<D, kShWarps>, (int)rows, kShThreads, 0, st, a, P, L, tc != nullptr)
                                 : sh_launch(k_shared_merge<D, 1>, (int)((rows + kShWarps - 1) / kShWarps), kShThreads, 0, st, a,
                                             P, L, tc != nullptr);
    return e == cudaSuccess ? BC_OK : BC_ERR_CUDA_BASE + (int)e;
}

bool sh_head_dim(int d) { return d == 32 || d == 64 || d == 128 || d == 256; }

// More query rows than this behind one prefix: the prefix kernel, else the rows kernel, which reads the
// prefix once per 8 rows.  Rows kernel against prefix kernel, 32 / 8 heads of 128: at 65536 keys 16 rows 59.3 /
// 83.8 us, 24 rows 82.9 / 86.0, 32 rows 105.1 / 85.8; 24 rows at 8192 keys 23.0 / 31.4, at 200000 221.8 / 192.3;
// at 65536 24 rows of heads of 64 60.2 / 74.9, without codes 50.7 / 67.8.  (Lengths are on the device: 32 rows
// behind 1000 keys, 14.2 / 20.0, pay for those behind long prefixes.)
constexpr int kShTcRows = 24;
bool sh_takes_tc(int n_seqs, int n_groups, int group, int head_dim) {
    return (head_dim == 64 || head_dim == 128) && (int64_t)(n_seqs / n_groups) * group > kShTcRows && n_seqs > n_groups;
}

ShList sh_list(int n_seqs, int n_groups, int group, bool prefixes) {
    ShList L{};
    const int64_t shared = (int64_t)(n_seqs / n_groups) * group;
    L.n_pre = prefixes ? n_groups : 0;
    L.n_own = n_seqs;
    L.pre_blocks = (int)((shared + kShRows - 1) / kShRows);
    L.own_blocks = (group + kShRows - 1) / kShRows;
    L.shift = 5;
    L.rows = kShRows;
    L.copies = 1;
    L.cost = kShItemCost;
    return L;
}

size_t sh_bytes(const ShList& L, int n_kv, int max_workers, int d) {
    return (size_t)(sh_first_item(L, n_kv, L.n_pre + L.n_own) + max_workers) * L.copies * L.rows * (d + 4) * sizeof(float);
}

}  // namespace
}  // namespace bc

using namespace bc;

extern "C" {

size_t bc_decode_shared_workspace_bytes(int n_seqs, int n_groups, int n_kv_heads, int group, int head_dim) {
    if (n_seqs <= 0 || n_groups <= 0 || n_seqs % n_groups || n_kv_heads <= 0 || group <= 0 || !sh_head_dim(head_dim))
        return 0;
    const bool tc = sh_takes_tc(n_seqs, n_groups, group, head_dim);
    return sh_bytes(sh_list(n_seqs, n_groups, group, !tc), n_kv_heads, kShMaxWorkers, head_dim) +
           (tc ? sh_bytes(sh_tc_list(n_seqs, n_groups, group), n_kv_heads, kShTcWorkers, head_dim) +
                     sh_tc_scratch((int64_t)n_seqs * n_kv_heads * group, head_dim)
               : 0);
}

int bc_decode_attention_shared(const void* q, bc_kv_planes K, bc_kv_planes V, bc_page_table pt,
                               const int32_t* seq_lens, const int32_t* prefix_lens, void* out, int n_seqs,
                               int n_groups, int n_kv_heads, int group, int head_dim, int mode, void* workspace,
                               size_t workspace_bytes, void* stream) {
    if (!bc_valid_head_dim(head_dim)) return BC_ERR_HEAD_DIM;
    if (!sh_head_dim(head_dim)) return BC_ERR_UNSUPPORTED;
    if (n_seqs < 0 || n_kv_heads <= 0 || group <= 0) return BC_ERR_ARG;
    if (mode != BC_MODE_BINARY && mode != BC_MODE_COMPENSATED) return BC_ERR_ARG;
    if (n_seqs == 0) return BC_OK;
    if (n_groups <= 0 || n_seqs % n_groups) return BC_ERR_ARG;
    if ((int64_t)n_seqs * n_kv_heads > INT32_MAX / group) return BC_ERR_TOO_LARGE;
    if (!q || !out || !seq_lens) return BC_ERR_ARG;
    if (!pt.pages || pt.page_size <= 0 || pt.page_size % 128 != 0 || pt.n_pages <= 0 || pt.max_pages <= 0)
        return BC_ERR_ARG;
    const bool comp = mode == BC_MODE_COMPENSATED;
    const void* planes[8] = {K.sign, K.bscale, V.sign, V.bscale, K.nib, K.rscale, V.nib, V.rscale};
    for (int i = 0; i < (comp ? 8 : 4); ++i) {
        if (!planes[i]) return BC_ERR_ARG;
        if (!bc_aligned(planes[i], 16)) return BC_ERR_ALIGN;
    }
    if (!bc_aligned(q, 2) || !bc_aligned(out, 2) || !bc_aligned(seq_lens, 4) || !bc_aligned(prefix_lens, 4) ||
        !bc_aligned(pt.pages, 4) || !bc_aligned(workspace, 16))
        return BC_ERR_ALIGN;
    if (!workspace ||
        workspace_bytes < bc_decode_shared_workspace_bytes(n_seqs, n_groups, n_kv_heads, group, head_dim))
        return BC_ERR_WORKSPACE;
    SharedArgs a{};
    a.q = (const __half*)q;
    a.q_aligned = bc_aligned(q, 16);
    a.K = K;
    a.V = V;
    a.pt = pt;
    a.seq_lens = seq_lens;
    a.prefix_lens = prefix_lens;
    a.out = (__half*)out;
    a.err = bc_device_error_ptr();
    if (!a.err) return BC_ERR_CUDA_BASE;
    a.n_seqs = n_seqs;
    a.n_groups = n_groups;
    a.per = n_seqs / n_groups;
    a.n_kv = n_kv_heads;
    a.group = group;
    const bool tc = sh_takes_tc(n_seqs, n_groups, group, head_dim) && prefix_lens;
    ShList L = sh_list(n_seqs, n_groups, group, !tc), T = sh_tc_list(n_seqs, n_groups, group);
    L.records = (float*)workspace;
    void* scratch = nullptr;
    if (tc) {
        T.n_workers = kShTcWorkers;
        T.records = (float*)((char*)workspace + sh_bytes(L, n_kv_heads, kShMaxWorkers, head_dim));
        scratch = (char*)T.records + sh_bytes(T, n_kv_heads, kShTcWorkers, head_dim);
    }
    cudaStream_t st = (cudaStream_t)stream;
    const ShList* t = tc ? &T : nullptr;
    switch (head_dim) {
        case 32: return comp ? sh_run<32, true>(a, L, t, scratch, st) : sh_run<32, false>(a, L, t, scratch, st);
        case 64: return comp ? sh_run<64, true>(a, L, t, scratch, st) : sh_run<64, false>(a, L, t, scratch, st);
        case 128: return comp ? sh_run<128, true>(a, L, t, scratch, st) : sh_run<128, false>(a, L, t, scratch, st);
        default: return comp ? sh_run<256, true>(a, L, t, scratch, st) : sh_run<256, false>(a, L, t, scratch, st);
    }
}

}  // extern "C"
