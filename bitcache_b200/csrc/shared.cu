// Decode attention of a batch over a paged cache whose sequences share
// prefixes: positions [0, prefix) of a group of sequences are read once for all
// of the group's query heads, the rest once per sequence.  Ragged lengths, held
// in device memory.  sm_100a.
//
// Mathematics (as bc_decode_attention), query row q, key with sign bits k, codes
// n and scales bs, rs, value likewise:
//   s   = (bs mean|q| (sgn q . sgn k) + rs / 7 (q . n)) / sqrt(d)
//   out = sum_s softmax(s) (bs_v sgn v + rs_v / 7 n_v)
// Work is a flat list of units, one unit being one 128-key tile for one block of
// up to 8 query rows of one kv head ("item": a prefix of a group, or the rest of
// a sequence).  The grid divides the list evenly, so ragged lengths need no plan
// on the host; a CTA's stretch of an item is a piece, whose record (U, l, o)
// k_shared_merge joins with the row's other pieces.
//
// Rows are the narrow side of every product (mma.sync m16n8k16, fp16 in, fp32
// accumulators): the 16 rows of A are keys in the scores and dims in the values,
// the 8 columns of B are query rows.  A is built in registers from the packed
// bytes, two instructions per pair of elements and no scale: sign bits become
// +-1, codes n become the fp16 numbers 24 + n (the nibble n + 8 in the mantissa
// of 16), whose constant part 24 sum(b) is subtracted at the end.  A key's
// scales multiply its few scores, and its probabilities before they become the
// value product's B operand: P1 = e bs, P2 = e rs / 7, rounded to fp16.  They
// keep at least 11 significant bits down to 2^-22 of a row's largest one: e is
// 2^(s - U) with U such that the largest P lies between 2^8 and 2^15.
#include "common.cuh"

namespace bc {
namespace {

constexpr int kShThreads = 128;
constexpr int kShWarps = kShThreads / 32;
constexpr int kShTile = 128;   // keys per unit: 32 per warp
constexpr int kShRows = 8;     // query rows per unit
constexpr int kShStages = 2;
constexpr int kShMaxCtas = 148 * 8;  // bound of the grid, for the workspace's size
constexpr float kShLog2e = 1.4426950408889634f;
constexpr float kShNone = -1e30f;  // U of a row without keys

struct SharedArgs {
    const __half* q;
    bc_kv_planes K, V;
    bc_page_table pt;
    const int32_t* seq_lens;
    const int32_t* prefix_lens;  // null: no prefixes
    __half* out;
    float* ws;
    unsigned int* err;
    int n_seqs, n_groups, per;  // per: sequences of a group
    int n_kv, group;
    int prefix_blocks, own_blocks;  // blocks of 8 query rows of a prefix item / of a sequence's own item
    int n_ctas;
};

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
    static constexpr int STAGE_B = 2 * HALF_B;
    static constexpr int MG_B = 2 * kShRows * (D + 4) * 4;  // two warps' records
    static constexpr int Q_OFF = kShStages * STAGE_B;
    static constexpr int Q_B = kShRows * (D + 8) * 2;
    static constexpr int MG_OFF = Q_OFF + Q_B;
    static constexpr int SCAN_OFF = MG_OFF + MG_B;
    static constexpr int SCAN_B = (kShThreads + 1) * 8 + 32;
    static constexpr int BAR_OFF = (SCAN_OFF + SCAN_B + 15) / 16 * 16;
    static constexpr int SMEM_B = BAR_OFF + 2 * kShStages * 8 + kShStages * 4 + 16 + 128;
};

__host__ __device__ constexpr int sh_record_floats(int d) { return kShRows * (d + 4); }

// ---- the list of work ------------------------------------------------------
__device__ __forceinline__ int sh_capacity(const SharedArgs& a) {
    const int64_t c = (int64_t)a.pt.max_pages * a.pt.page_size;
    return (int)(c < 0x7fffff80 ? c : 0x7fffff80);
}
__device__ __forceinline__ int sh_len(const SharedArgs& a, int b) {
    return max(0, min(__ldg(a.seq_lens + b), sh_capacity(a)));
}
// A group of one sequence shares with nobody: its prefix is part of its own keys.
__device__ __forceinline__ int sh_prefix(const SharedArgs& a, int g) {
    if (!a.prefix_lens || a.per == 1) return 0;
    return max(0, min(__ldg(a.prefix_lens + g), sh_capacity(a)));
}

// Entry e of the list: group e's prefix (e < n_groups), else sequence e - n_groups's own keys.
struct ShEntry {
    int lo, hi;  // key positions
    int tile0, tiles;
    int blocks;
};
__device__ __forceinline__ ShEntry sh_entry(const SharedArgs& a, int e) {
    ShEntry x;
    if (e < a.n_groups) {
        x.lo = 0;
        x.hi = sh_prefix(a, e);
        x.blocks = a.prefix_blocks;
    } else {
        const int b = e - a.n_groups;
        x.lo = sh_prefix(a, b / a.per);
        x.hi = sh_len(a, b);
        x.blocks = a.own_blocks;
    }
    x.tile0 = x.lo / kShTile;
    x.tiles = x.hi > x.lo ? (x.hi + kShTile - 1) / kShTile - x.tile0 : 0;
    return x;
}
__device__ __forceinline__ int64_t sh_units(const SharedArgs& a, const ShEntry& x) {
    return (int64_t)x.tiles * x.blocks * a.n_kv;
}
__device__ __forceinline__ int64_t sh_first_item(const SharedArgs& a, int e) {
    return e < a.n_groups ? (int64_t)e * a.n_kv * a.prefix_blocks
                          : (int64_t)a.n_groups * a.n_kv * a.prefix_blocks +
                                (int64_t)(e - a.n_groups) * a.n_kv * a.own_blocks;
}

// Exclusive sums of the entries' units over the CTA's threads (each thread a
// run of consecutive entries) in scan[0 .. kShThreads]; scan[kShThreads] is the total.
__device__ __forceinline__ int64_t sh_scan(const SharedArgs& a, int64_t* scan) {
    const int n = a.n_groups + a.n_seqs, chunk = (n + kShThreads - 1) / kShThreads;
    const int lane = threadIdx.x & 31;
    int64_t sum = 0;
    for (int e = threadIdx.x * chunk; e < min(n, ((int)threadIdx.x + 1) * chunk); ++e) sum += sh_units(a, sh_entry(a, e));
    scan[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        int64_t v[4], run = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = run;
            run += scan[4 * lane + i];
        }
        int64_t before = run;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, before, off);
            if (lane >= off) before += up;
        }
        if (lane == 31) scan[kShThreads] = before;
        before -= run;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) scan[4 * lane + i] = before + v[i];
    }
    __syncthreads();
    return scan[kShThreads];
}
static_assert(kShThreads == 128, "sh_scan: four sums per lane");

// CTA c's units: [sh_begin(c), sh_begin(c + 1)), n = min(CTAs, units) so that
// none of the n is empty.  A piece's record is number item + CTA: along the list
// every new piece raises one of the two.
__device__ __forceinline__ int64_t sh_begin(int64_t units, int n, int64_t c) { return units * c / n; }
__device__ __forceinline__ int sh_cta_of(int64_t units, int n, int64_t u) {
    return (int)(((u + 1) * n + units - 1) / units) - 1;
}

// Position in the list; every thread keeps its own copy.
struct ShCursor {
    int e;
    ShEntry x;
    int h, blk, tile;  // tile: index within the item
};
__device__ __forceinline__ void sh_seek(const SharedArgs& a, ShCursor& c, int e, int64_t at) {
    c.e = e;
    c.x = sh_entry(a, e);
    c.tile = (int)(at % c.x.tiles);
    const int64_t it = at / c.x.tiles;
    c.blk = (int)(it % c.x.blocks);
    c.h = (int)(it / c.x.blocks);
}
// Next unit; true when it begins another item.  Never called on the last unit.
__device__ __forceinline__ bool sh_next(const SharedArgs& a, ShCursor& c) {
    if (++c.tile < c.x.tiles) return false;
    c.tile = 0;
    if (++c.blk < c.x.blocks) return true;
    c.blk = 0;
    if (++c.h < a.n_kv) return true;
    c.h = 0;
    do c.x = sh_entry(a, ++c.e);
    while (c.x.tiles == 0);
    return true;
}

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
                 : "r"(smem_u32(row)));
}
// Two 16x16 byte matrices, transposed: lanes 0-15 / 16-31 give the rows of the
// first / second; lane (g, q) gets bytes g and g + 8 of rows 4q .. 4q + 3.
__device__ __forceinline__ void sh_ldsm_t2(const uint8_t* row, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(row)));
}
__device__ __forceinline__ void sh_ldsm_t1(const uint8_t* row, uint32_t& r0, uint32_t& r1) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x1.trans.shared.b8 {%0,%1}, [%2];"
                 : "=r"(r0), "=r"(r1)
                 : "r"(smem_u32(row)));
}
// Bits i and i + 16 of w as +-1 (1 for a set bit).
__device__ __forceinline__ uint32_t pm1(uint32_t w, int left) { return ((w << left) & 0x80008000u) ^ 0xBC00BC00u; }
// Nibbles at bits 0-3 and 16-19 of (w shifted) as 16 + u = 24 + code.
__device__ __forceinline__ uint32_t code24_l(uint32_t w, int left) { return ((w << left) & 0x03C003C0u) | 0x4C004C00u; }
__device__ __forceinline__ uint32_t code24_r(uint32_t w, int right) { return ((w >> right) & 0x03C003C0u) | 0x4C004C00u; }
// Nibbles t and t + 4 (t < 4).
__device__ __forceinline__ uint32_t code24(uint32_t w, int t) { return t < 2 ? code24_l(w, 6 - 4 * t) : code24_r(w, 4 * t - 6); }

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The query rows as B operands, and what the scores need of each row.
template <int D, bool COMP>
struct ShQuery {
    uint32_t sign[D / 16][2];
    uint32_t code[COMP ? D / 16 : 1][2];
    float bco[2], rco[2], off[2];  // rows 2q, 2q + 1: score = bs bco D1 + rs rco (D2 - off)
};

// Dim of element `half` (0, 1) of register r of k step s in the sign part / code part, lane column q.
template <int D>
__device__ __forceinline__ int sign_dim(int s, int r, int half, int q) {
    const int p = 2 * s + r;  // pair within the lane's D / 8
    if constexpr (D >= 128) return 32 * (q + 4 * (p / 16)) + p % 16 + 16 * half;
    if constexpr (D == 64) return 32 * (q / 2) + 8 * (q % 2) + p + 16 * half;
    return 4 * q + p + 16 * half;  // D == 32
}
template <int D>
__device__ __forceinline__ int code_dim(int s, int r, int half, int q) {
    const int c = s / 2, n = 2 * (s % 2) + r + 4 * half;  // chunk, nibble of its word q
    return nib_dim(D, c, 4 * q + n / 2, n % 2);
}

template <int D, bool COMP>
__device__ __forceinline__ void sh_load_query(const SharedArgs& a, const ShCursor& c, uint8_t* smem,
                                              ShQuery<D, COMP>& Q, int (&hi)[2], int& hi_min) {
    using C = ShCfg<D, COMP>;
    constexpr int ROW = D + 8;
    __half* qs = reinterpret_cast<__half*>(smem + C::Q_OFF);
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
    const bool prefix = c.e < a.n_groups;
    const int rows = prefix ? a.per * a.group : a.group;
    const int b0 = prefix ? c.e * a.per : c.e - a.n_groups;
    __syncthreads();  // the previous item's rows are read
    for (int i = threadIdx.x; i < kShRows * D; i += kShThreads) {
        const int r = c.blk * kShRows + i / D;
        __half v = __float2half(0.0f);
        if (r < rows)
            v = a.q[((int64_t)(b0 + r / a.group) * a.n_kv * a.group + (int64_t)c.h * a.group + r % a.group) * D + i % D];
        qs[(i / D) * ROW + i % D] = v;
    }
    __syncthreads();
    const __half* row = qs + g8 * ROW;
    float sum = 0.0f, mag = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const __half x0 = row[sign_dim<D>(s, r, 0, q)], x1 = row[sign_dim<D>(s, r, 1, q)];
            const float f0 = __half2float(x0), f1 = __half2float(x1);
            Q.sign[s][r] = (f0 >= 0.0f ? 0x3C00u : 0xBC00u) | (f1 >= 0.0f ? 0x3C000000u : 0xBC000000u);
            mag += fabsf(f0) + fabsf(f1);
            sum += f0 + f1;
            if constexpr (COMP) {
                const uint32_t y0 = __half_as_ushort(row[code_dim<D>(s, r, 0, q)]);
                const uint32_t y1 = __half_as_ushort(row[code_dim<D>(s, r, 1, q)]);
                Q.code[s][r] = y0 | (y1 << 16);
            }
        }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        mag += __shfl_xor_sync(0xffffffffu, mag, o);
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float scale = kShLog2e * rsqrtf((float)D);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float m = __shfl_sync(0xffffffffu, mag, 4 * (2 * q + j));
        const float t = __shfl_sync(0xffffffffu, sum, 4 * (2 * q + j));
        Q.bco[j] = m * (1.0f / D) * scale;
        Q.rco[j] = scale * (1.0f / 7.0f);
        Q.off[j] = 24.0f * t;
        const int r = c.blk * kShRows + 2 * q + j;
        // a sequence shorter than its group's prefix sees its own length of it
        hi[j] = prefix && r < rows ? min(c.x.hi, sh_len(a, b0 + r / a.group)) : c.x.hi;
    }
    hi_min = (int)__reduce_min_sync(0xffffffffu, (unsigned)min(hi[0], hi[1]));
}

// Accumulators of one warp: o[mt][4] with rows of m-tile mt = 2c + h the dims
// nib_dim(D, c, g8 (+ 8), h), columns the query rows 2q, 2q + 1.
template <int D>
struct ShState {
    float o[D / 16][4];
    float U[2], l[2], t[2];  // per row 2q, 2q + 1: unit, partial sums of e and of P2 over this lane's keys
};
template <int D>
__device__ __forceinline__ void sh_clear(ShState<D>& st) {
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[m][i] = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        st.U[j] = kShNone;
        st.l[j] = st.t[j] = 0.0f;
    }
}

// Position of matrix row r (0 .. 15) of a transposing load among its 16 keys:
// bytes 0, 2 of a lane's register are the k elements 2q, 2q + 1 and bytes 1, 3
// the elements 2q + 8, 2q + 9.
__device__ __forceinline__ int sh_key_of_row(int r) { return 2 * (r >> 2) + ((r >> 1) & 1) + 8 * (r & 1); }

// One warp's 32 keys (k0 .. k0 + 31 of the tile at key position kpos) of a stage.
template <int D, bool COMP>
__device__ __forceinline__ void sh_consume(const ShQuery<D, COMP>& Q, ShState<D>& st, const uint8_t* sb, int k0,
                                           int kpos, int lo, const int (&hi)[2], bool masked) {
    using C = ShCfg<D, COMP>;
    constexpr int NW = C::NW;
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
    const uint8_t *ks = sb, *vs = sb + C::HALF_B;
    float s[2][4];
    // ---- scores of two blocks of 16 keys
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int kb = k0 + 16 * b;
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
            for (int st2 = 0; st2 < PAIRS / 2; ++st2) {
                const int p = 2 * st2;
                mma_f16(d1, pm1(w[0][p / 16], 15 - p % 16), pm1(w[1][p / 16], 15 - p % 16),
                        pm1(w[0][p / 16], 14 - p % 16), pm1(w[1][p / 16], 14 - p % 16), Q.sign[st2][0],
                        Q.sign[st2][1]);
            }
        }
        if constexpr (COMP) {
            const uint8_t* nib = ks + C::NIB_OFF + (kb >> 3) * 4 * D;
            // word q of chunk c of key g8 (blk 0) and g8 + 8 (blk 1)
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
            for (int c = 0; c < NW; ++c)
#pragma unroll
                for (int t = 0; t < 4; t += 2)
                    mma_f16(d2, code24(n[c][0], t), code24(n[c][1], t), code24(n[c][0], t + 1), code24(n[c][1], t + 1),
                            Q.code[2 * c + t / 2][0], Q.code[2 * c + t / 2][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int key = kb + g8 + 8 * x;
            const float bs = __half2float(reinterpret_cast<const __half*>(ks + C::BS_OFF)[key]);
            const float rs = COMP ? __half2float(reinterpret_cast<const __half*>(ks + C::RS_OFF)[key]) : 0.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float v = bs * (Q.bco[j] * d1[2 * x + j]);
                if constexpr (COMP) v += rs * (Q.rco[j] * (d2[2 * x + j] - Q.off[j]));
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
            const int key = k0 + 16 * b + g8 + 8 * x;
            vb[b][x] = __half2float(reinterpret_cast<const __half*>(vs + C::BS_OFF)[key]);
            vr[b][x] = COMP ? __half2float(reinterpret_cast<const __half*>(vs + C::RS_OFF)[key]) * (1.0f / 7.0f) : 0.0f;
            // 2^grow bounds the larger scale; a key whose scales are next to 0 does not pull U down by more than 2^40
            const float grow = (float)max(-40, (__float_as_int(fmaxf(vb[b][x], vr[b][x])) >> 23) - 126);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float& v = s[b][2 * x + j];
                if (masked && (kpos + key < lo || kpos + key >= hi[j])) v = -INFINITY;
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
            st.t[j] *= f;
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
            float e[2], c1[2], c2[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float v = s[b][2 * x + j];
                e[j] = exp2f(v - st.U[j]);
                st.l[j] += e[j];
                const bool out = masked && v == -INFINITY;  // a masked row's scales may be anything
                c1[j] = out ? 0.0f : e[j] * vb[b][x];
                c2[j] = out ? 0.0f : e[j] * vr[b][x];
            }
            p1[x] = pack_h2(c1[0], c1[1]);
            if constexpr (COMP) {
                p2[x] = pack_h2(c2[0], c2[1]);
                const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&p2[x]));
                st.t[0] += r.x;
                st.t[1] += r.y;
                p2[x] = movmatrix(p2[x]);
            }
            p1[x] = movmatrix(p1[x]);
        }
        const int kb = k0 + 16 * b;
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
                wd[i] = reinterpret_cast<const uint32_t*>(vs)[kb + sh_key_of_row(4 * q + i)];
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
                        a0 = pm1(sg[2 * w], 15 - t);
                        a1 = pm1(sg[2 * w + 1], 15 - t);
                        a2 = pm1(sg[2 * w], 7 - t);
                        a3 = pm1(sg[2 * w + 1], 7 - t);
                    } else if constexpr (D == 64) {
                        const int t = 2 * (c + cx) + 4 * h;
                        a0 = pm1(sg[0], 15 - t);
                        a1 = pm1(sg[0], 14 - t);
                        a2 = pm1(sg[0], 7 - t);
                        a3 = pm1(sg[0], 6 - t);
                    } else {
                        const int left = 15 - 2 * g8 - h;
                        a0 = pm1(__byte_perm(wd[0], wd[2], 0x5410), left);
                        a1 = pm1(__byte_perm(wd[0], wd[2], 0x7632), left);
                        a2 = pm1(__byte_perm(wd[1], wd[3], 0x5410), left);
                        a3 = pm1(__byte_perm(wd[1], wd[3], 0x7632), left);
                    }
                    mma_f16(o, a0, a1, a2, a3, p1[0], p1[1]);
                    if constexpr (COMP) {
                        const uint32_t x0 = r[2 * cx], x1 = r[2 * cx + 1];
                        if (h == 0)
                            mma_f16(o, code24_l(x0, 6), code24_l(x1, 6), code24_r(x0, 2), code24_r(x1, 2), p2[0], p2[1]);
                        else
                            mma_f16(o, code24_l(x0, 2), code24_l(x1, 2), code24_r(x0, 6), code24_r(x1, 6), p2[0], p2[1]);
                    }
                }
        }
    }
}

// Join the four warps' sums and write the piece's record:
// floats [8 rows][D] o, then [8 rows][2] (U, l).
template <int D, bool COMP>
__device__ __forceinline__ void sh_flush(const SharedArgs& a, ShState<D>& st, uint8_t* smem, int64_t record) {
    using C = ShCfg<D, COMP>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2, q = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            st.l[j] += __shfl_xor_sync(0xffffffffu, st.l[j], o);
            st.t[j] += __shfl_xor_sync(0xffffffffu, st.t[j], o);
        }
        if constexpr (COMP) {
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
                st.o[mt][j] -= 24.0f * st.t[j];
                st.o[mt][2 + j] -= 24.0f * st.t[j];
            }
        }
    }
    constexpr int REC = kShRows * (D + 4);
    auto put = [&](float* m) {  // [2q + j][dim], rows D + 4 floats apart; (U, l) behind each row
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float* row = m + (2 * q + j) * (D + 4);
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
                row[nib_dim(D, mt / 2, g8, mt % 2)] = st.o[mt][j];
                row[nib_dim(D, mt / 2, g8 + 8, mt % 2)] = st.o[mt][2 + j];
            }
            if (g8 == 0) {
                row[D] = st.U[j];
                row[D + 1] = st.l[j];
            }
        }
    };
    auto add = [&](const float* m) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float* row = m + (2 * q + j) * (D + 4);
            const float U = fmaxf(st.U[j], row[D]), f = exp2f(st.U[j] - U), g = exp2f(row[D] - U);
            st.U[j] = U;
            st.l[j] = st.l[j] * f + row[D + 1] * g;
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
                st.o[mt][j] = st.o[mt][j] * f + row[nib_dim(D, mt / 2, g8, mt % 2)] * g;
                st.o[mt][2 + j] = st.o[mt][2 + j] * f + row[nib_dim(D, mt / 2, g8 + 8, mt % 2)] * g;
            }
        }
    };
    float* mg = reinterpret_cast<float*>(smem + C::MG_OFF);
    if (warp >= 2) put(mg + (warp - 2) * REC);
    __syncthreads();
    if (warp < 2) add(mg + warp * REC);
    __syncthreads();
    if (warp == 1) put(mg);
    __syncthreads();
    if (warp == 0) {
        add(mg);
        put(a.ws + record * REC);
    }
}

__device__ __forceinline__ void sh_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <int D, bool COMP>
__global__ void __launch_bounds__(kShThreads) k_shared_rows(const SharedArgs a) {
    using C = ShCfg<D, COMP>;
    extern __shared__ __align__(128) uint8_t sh_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sh_raw) + 127) & ~uintptr_t(127));
    int64_t* scan = reinterpret_cast<int64_t*>(smem + C::SCAN_OFF);
    int64_t* found = scan + kShThreads + 1;  // entry and unit within it of the CTA's first unit
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    uint64_t* empty = full + kShStages;
    int* present = reinterpret_cast<int*>(empty + kShStages);  // per stage: its page is in the pool
    const int tid = threadIdx.x, warp = tid >> 5;

    if (tid == 0) {
        for (int s = 0; s < kShStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kShWarps);
        }
        fence_mbar_init();
    }
    const int64_t units = sh_scan(a, scan);
    const int n_ctas = (int)min((int64_t)a.n_ctas, units);
    if (blockIdx.x == 0) {  // lengths outside the block table are cut, and said so
        const int64_t cap = (int64_t)a.pt.max_pages * a.pt.page_size;
        for (int b = tid; b < a.n_seqs; b += kShThreads)
            if (a.seq_lens[b] < 0 || a.seq_lens[b] > cap) raise_device_error(a.err, BC_DEVERR_INDEX);
        if (a.prefix_lens)
            for (int g = tid; g < a.n_groups; g += kShThreads)
                if (a.prefix_lens[g] < 0 || a.prefix_lens[g] > cap) raise_device_error(a.err, BC_DEVERR_INDEX);
    }
    if ((int)blockIdx.x >= n_ctas) return;
    const int64_t u0 = sh_begin(units, n_ctas, blockIdx.x), u1 = sh_begin(units, n_ctas, blockIdx.x + 1);
    if (scan[tid] <= u0 && u0 < scan[tid + 1]) {
        const int n = a.n_groups + a.n_seqs, chunk = (n + kShThreads - 1) / kShThreads;
        int64_t at = u0 - scan[tid];
        int e = tid * chunk;
        for (;; ++e) {
            const int64_t w = sh_units(a, sh_entry(a, e));
            if (at < w) break;
            at -= w;
        }
        found[0] = e;
        found[1] = at;
    }
    __syncthreads();
    ShCursor cur, ahead;
    sh_seek(a, cur, (int)found[0], found[1]);
    ahead = cur;

    const int n_units = (int)(u1 - u0);
    auto issue = [&](int it) {  // thread 0: the tile `ahead` points at, into stage it % kShStages
        const int s = it % kShStages;
        uint8_t* dst = smem + s * C::STAGE_B;
        const int seq = ahead.e < a.n_groups ? ahead.e * a.per : ahead.e - a.n_groups;
        const int64_t pos = (int64_t)(ahead.x.tile0 + ahead.tile) * kShTile;
        const int pg = __ldg(a.pt.pages + ((int64_t)seq * a.n_kv + ahead.h) * a.pt.max_pages + pos / a.pt.page_size);
        const bool ok = pg >= 0 && pg < a.pt.n_pages;
        present[s] = ok;
        if (!ok) {
            raise_device_error(a.err, BC_DEVERR_PAGE);
            sh_arrive(&full[s]);
            return;
        }
        const int64_t row = (int64_t)pg * a.pt.page_size + pos % a.pt.page_size;
        mbar_arrive_expect_tx(&full[s], C::STAGE_B);
        auto part = [&](const bc_kv_planes& P, uint8_t* d) {
            bulk_g2s(d, (const uint8_t*)P.sign + row * (D / 8), C::SIGN_B, &full[s]);
            bulk_g2s(d + C::BS_OFF, (const uint8_t*)P.bscale + row * 2, C::SC_B, &full[s]);
            if constexpr (COMP) {
                bulk_g2s(d + C::NIB_OFF, (const uint8_t*)P.nib + row * (D / 2), C::NIB_B, &full[s]);
                bulk_g2s(d + C::RS_OFF, (const uint8_t*)P.rscale + row * 2, C::SC_B, &full[s]);
            }
        };
        part(a.K, dst);
        part(a.V, dst + C::HALF_B);
    };
    int issued = 0;
    if (tid == 0)
        for (; issued < min(kShStages, n_units); ++issued) {
            if (issued) sh_next(a, ahead);
            issue(issued);
        }

    ShQuery<D, COMP> Q;
    ShState<D> st;
    int hi[2], hi_min;
    sh_load_query<D, COMP>(a, cur, smem, Q, hi, hi_min);
    sh_clear(st);
    bool alive = true;
    for (int it = 0; it < n_units; ++it) {
        const int s = it % kShStages;
        const uint32_t phase = (uint32_t)(it / kShStages) & 1u;
        if (it > 0 && sh_next(a, cur)) {
            sh_load_query<D, COMP>(a, cur, smem, Q, hi, hi_min);
            sh_clear(st);
        }
        // refill the stage that the previous unit left, once all warps have
        if (tid == 0 && it > 0 && issued < n_units) {
            const int ps = (it - 1) % kShStages;
            if (alive && mbar_wait_bounded(&empty[ps], (uint32_t)((it - 1) / kShStages) & 1u)) {
                fence_proxy_async_smem();
                sh_next(a, ahead);
                issue(issued++);
            } else if (alive) {
                raise_device_error(a.err, BC_DEVERR_TIMEOUT);
                alive = false;
            }
        }
        alive = __all_sync(0xffffffffu, alive);
        alive = __all_sync(0xffffffffu, alive && mbar_wait_bounded(&full[s], phase));
        if (alive) {
            const int kpos = (cur.x.tile0 + cur.tile) * kShTile;
            const bool here = present[s] != 0;
            if (here)
                sh_consume<D, COMP>(Q, st, smem + s * C::STAGE_B, 32 * warp, kpos, cur.x.lo, hi,
                                    kpos < cur.x.lo || kpos + kShTile > hi_min);
        } else if ((tid & 31) == 0) {
            raise_device_error(a.err, BC_DEVERR_TIMEOUT);
        }
        __syncwarp();
        if ((tid & 31) == 0) sh_arrive(&empty[s]);
        const bool last = it + 1 == n_units || cur.tile + 1 == cur.x.tiles;
        if (last) {
            const int64_t item = sh_first_item(a, cur.e) + (int64_t)cur.h * cur.x.blocks + cur.blk;
            sh_flush<D, COMP>(a, st, smem, item + blockIdx.x);
        }
    }
    if (!alive && tid == 0)  // gave up: let the copies in flight land (bounded) before the memory is reused
        for (int i = max(0, issued - kShStages); i < issued; ++i)
            mbar_wait_bounded(&full[i % kShStages], (uint32_t)(i / kShStages) & 1u);
}

// One CTA per (sequence, kv head): joins the pieces of each query row.
template <int D>
__global__ void __launch_bounds__(kShThreads) k_shared_merge(const SharedArgs a) {
    constexpr int REC = kShRows * (D + 4), PER = D / 32;
    __shared__ int64_t scan[kShThreads + 1], at[2];
    const int b = blockIdx.x / a.n_kv, h = blockIdx.x % a.n_kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t units = sh_scan(a, scan);
    const int n_ctas = (int)min((int64_t)a.n_ctas, units);
    const int n = a.n_groups + a.n_seqs, chunk = (n + kShThreads - 1) / kShThreads;
    const int want[2] = {b / a.per, a.n_groups + b};
    ShEntry x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if ((int)threadIdx.x == want[i] / chunk) {
            int64_t sum = scan[threadIdx.x];
            for (int e = threadIdx.x * chunk; e < want[i]; ++e) sum += sh_units(a, sh_entry(a, e));
            at[i] = sum;
        }
        x[i] = sh_entry(a, want[i]);
    }
    __syncthreads();
    for (int g = warp; g < a.group; g += kShWarps) {
        const int64_t head = ((int64_t)b * a.n_kv + h) * a.group + g;
        float M = kShNone, L = 0.0f, o[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (x[i].tiles == 0) continue;
            const int r = i == 0 ? (b % a.per) * a.group + g : g;
            const int64_t it = (int64_t)h * x[i].blocks + r / kShRows;
            const int64_t first = at[i] + it * x[i].tiles;
            const int c0 = sh_cta_of(units, n_ctas, first), c1 = sh_cta_of(units, n_ctas, first + x[i].tiles - 1);
            const float* rec = a.ws + (sh_first_item(a, want[i]) + it) * REC + (r % kShRows) * (D + 4);
            for (int c = c0; c <= c1; ++c) {
                const float* p = rec + (int64_t)c * REC;
                const float U = fmaxf(M, p[D]), f = exp2f(M - U), w = exp2f(p[D] - U);
                M = U;
                L = L * f + p[D + 1] * w;
#pragma unroll
                for (int k = 0; k < PER; ++k) o[k] = o[k] * f + p[32 * k + lane] * w;
            }
        }
        const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;  // no keys: zeros
#pragma unroll
        for (int k = 0; k < PER; ++k) a.out[head * D + 32 * k + lane] = __float2half_rn(o[k] * inv);
    }
}

template <int D, bool COMP>
int sh_ctas(int* n_ctas) {
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
        cached[dev] = min(sms * occ, kShMaxCtas);
    }
    *n_ctas = cached[dev];
    return BC_OK;
}

template <int D, bool COMP>
int sh_run(SharedArgs& a, cudaStream_t st) {
    const int rc = sh_ctas<D, COMP>(&a.n_ctas);
    if (rc) return rc;
    k_shared_rows<D, COMP><<<a.n_ctas, kShThreads, ShCfg<D, COMP>::SMEM_B, st>>>(a);
    BC_LAUNCH_CHECK();
    k_shared_merge<D><<<a.n_seqs * a.n_kv, kShThreads, 0, st>>>(a);
    BC_LAUNCH_CHECK();
    return BC_OK;
}

bool sh_head_dim(int d) { return d == 32 || d == 64 || d == 128 || d == 256; }

int64_t sh_records(int n_seqs, int n_groups, int n_kv, int group) {
    const int per = n_seqs / n_groups;
    const int64_t prefix = ((int64_t)per * group + kShRows - 1) / kShRows, own = (group + kShRows - 1) / kShRows;
    return (int64_t)n_groups * n_kv * prefix + (int64_t)n_seqs * n_kv * own + kShMaxCtas;
}

}  // namespace
}  // namespace bc

using namespace bc;

extern "C" {

size_t bc_decode_shared_workspace_bytes(int n_seqs, int n_groups, int n_kv_heads, int group, int head_dim) {
    if (n_seqs <= 0 || n_groups <= 0 || n_seqs % n_groups || n_kv_heads <= 0 || group <= 0 || !sh_head_dim(head_dim))
        return 0;
    return (size_t)sh_records(n_seqs, n_groups, n_kv_heads, group) * sh_record_floats(head_dim) * sizeof(float);
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
    if ((int64_t)n_seqs * n_kv_heads > INT32_MAX || (int64_t)n_seqs * group > INT32_MAX) return BC_ERR_TOO_LARGE;
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
    a.K = K;
    a.V = V;
    a.pt = pt;
    a.seq_lens = seq_lens;
    a.prefix_lens = prefix_lens;
    a.out = (__half*)out;
    a.ws = (float*)workspace;
    a.err = bc_device_error_ptr();
    if (!a.err) return BC_ERR_CUDA_BASE;
    a.n_seqs = n_seqs;
    a.n_groups = n_groups;
    a.per = n_seqs / n_groups;
    a.n_kv = n_kv_heads;
    a.group = group;
    a.prefix_blocks = (int)(((int64_t)a.per * group + kShRows - 1) / kShRows);
    a.own_blocks = (group + kShRows - 1) / kShRows;
    cudaStream_t st = (cudaStream_t)stream;
    switch (head_dim) {
        case 32: return comp ? sh_run<32, true>(a, st) : sh_run<32, false>(a, st);
        case 64: return comp ? sh_run<64, true>(a, st) : sh_run<64, false>(a, st);
        case 128: return comp ? sh_run<128, true>(a, st) : sh_run<128, false>(a, st);
        default: return comp ? sh_run<256, true>(a, st) : sh_run<256, false>(a, st);
    }
}

}  // extern "C"
