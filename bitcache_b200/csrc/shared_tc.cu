// The prefix part of bc_decode_attention_shared when many query rows share a
// prefix: S = Q K^T and O += P V on the 5th-generation tensor cores.  sm_100a.
//
// An item is a block of up to 128 query rows of one kv head (M = 128, one row per
// tensor-memory lane) against a prefix, in tiles of 128 keys (N of the scores, K
// of the values).  A score needs two dots, sgn q . sgn k and q . n, with scales of
// the key's own, so K holds both parts side by side, scaled, and Q likewise:
//   K = [ bs sgn k | rs / 8 n ],  Q = [ h sgn q | 8 / 7 q / f ],  h = fp16(mean|q|),
//   f = mean|q| / h:  s = f Q . K
// (f carries what the rounding of the row's mean would lose).  V = bs sgn v + rs/7 n.
//
// Roles of the 15 warps of a CTA, one CTA per SM:
//   0-3    softmax: a thread owns a query row.  Writes the row's Q into tensor
//          memory, then per tile reads its 128 scores, keeps U and l, writes P
//          (fp16, over the scores) and, when U moves, rescales O.
//   4-7    unpack K: a thread owns a key; packed bytes -> fp16 operand rows in
//          shared memory (128-byte swizzle, K-major: 4 blocks of 64 elements).
//   8-11   unpack V, likewise (MN-major: dims contiguous, 64 per swizzle atom).
//   12     issues the products: Q (tensor memory) x K, P (tensor memory) x V.
//   13, 14 bring K's / V's packed tiles with 1-D bulk copies, three ahead.
// Keeping Q in tensor memory spares half of the score product's shared-memory
// reads, which with the operands' own writes are what bounds the kernel: per
// tile 96 KB written, 96 KB read by the tensor cores and 43 KB of packed bytes in
// and out at 128 B per clock are 1900 clocks, the products 1536, the exponentials
// of 128 rows 1024, and the unpacking about 800 issue slots per scheduler.
//
// Scores are scaled so that P = 2^(s - U) lies below 2^15, U rising when it would
// not, to 2^8 above the largest; the elements of K, V, Q and P are rounded to fp16
// once each, sums are fp32.
#include "shared.cuh"
#include "shared_tc.h"

namespace bc {
namespace {

constexpr int kTcTile = 128;
constexpr int kTcThreads = 480;
constexpr int kTcRaw = 3;        // packed tiles ahead
constexpr int kTcItemCost = 2;   // an item's start and end, in tiles
constexpr uint32_t kTcSpin = 1u << 22;

template <int D, bool COMP>
struct TcCfg {
    static constexpr int KE = COMP ? 2 * D : D;              // elements of a K row
    static constexpr int KOP_B = kTcTile * KE * 2;
    static constexpr int VOP_B = kTcTile * D * 2;
    static constexpr int VST = D == 128 && COMP ? 1 : 2;     // V operand tiles
    static constexpr int SIGN_B = kTcTile * D / 8;
    static constexpr int NIB_B = COMP ? kTcTile * D / 2 : 0;
    static constexpr int SC_B = kTcTile * 2;
    static constexpr int BS_OFF = SIGN_B + NIB_B;
    static constexpr int RS_OFF = BS_OFF + SC_B;
    static constexpr int RAW_B = SIGN_B + NIB_B + SC_B * (COMP ? 2 : 1);
    static constexpr int V_OFF = 2 * KOP_B;
    static constexpr int RAWK_OFF = V_OFF + VST * VOP_B;
    static constexpr int RAWV_OFF = RAWK_OFF + kTcRaw * RAW_B;
    static constexpr int SCAN_OFF = (RAWV_OFF + kTcRaw * RAW_B + 15) / 16 * 16;
    static constexpr int BAR_OFF = SCAN_OFF + (kShThreads + 1) * 8 + 8;
    static constexpr int FLAG_OFF = BAR_OFF + 32 * 8;
    static constexpr int SMEM_B = FLAG_OFF + 20 * 4 + 1024;  // + alignment to the swizzle atom
    // tensor memory columns
    static constexpr int S_COL = 0, O_COL = 256, Q_COL = 256 + D;
    static_assert(Q_COL + KE / 2 <= 512, "tensor memory");
};

enum TcBar {
    kRawKFull = 0, kRawKEmpty = 3, kRawVFull = 6, kRawVEmpty = 9, kKFull = 12, kKEmpty = 14, kVFull = 16, kVEmpty = 18,
    kSFull = 20, kPFull = 22, kQFull = 24, kPvDone = 25, kDrain = 26, kTcBars = 27
};

// ---- tcgen05 ---------------------------------------------------------------
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: lane's row, one register per column.
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle.  Groups of 8 rows (K-major)
// or of 8 k (MN-major) are 1024 bytes apart; `lead` is the distance between the
// 64-element atoms of an MN-major operand.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// fp16 x fp16 -> fp32, M = 128; B K-major, or MN-major.
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n / 8) << 17) | (8u << 24);
}

// ---- waits -----------------------------------------------------------------
// Bounded; once one has given up (dead), all do, and the CTA winds down.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
    if (mbar_try_wait(bar, parity)) return true;
    for (uint32_t it = 0; it < kTcSpin; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
    }
    *dead = 1;
    return false;
}
__device__ __forceinline__ void tc_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
// Codes of nibbles t and t + 4 (t < 4) of w, exact: the nibble in the mantissa of 1024.
__device__ __forceinline__ __half2 tc_code(uint32_t w, int t) {
    const uint32_t x = t < 2 ? w : w >> 8;
    if (t % 2 == 0) return __hsub2(bits_h2((x & 0x000F000Fu) | 0x64006400u), bits_h2(0x64086408u));
    return __hfma2(bits_h2((x & 0x00F000F0u) | 0x64006400u), bits_h2(0x2C002C00u), bits_h2(0xD480D480u));  // /16 - 72
}
// +-s for bits i and i + 16 of w (flip = s with its sign set).
__device__ __forceinline__ uint32_t tc_sign(uint32_t w, int i, uint32_t flip) { return ((w << (15 - i)) & 0x80008000u) ^ flip; }
__device__ __forceinline__ void sts128(uint8_t* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(smem_u32(p)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

template <int D, bool COMP>
__global__ void __launch_bounds__(kTcThreads, 1) k_shared_prefix(const SharedArgs a, const ShList L) {
    using C = TcCfg<D, COMP>;
    constexpr int NW = D / 32;
    extern __shared__ uint8_t tc_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    int64_t* scan = reinterpret_cast<int64_t*>(smem + C::SCAN_OFF);
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    volatile int* flags = reinterpret_cast<volatile int*>(smem + C::FLAG_OFF);
    volatile int* kbad = flags;        // [8] tile i % 8: its page is outside the pool
    volatile int* vbad = flags + 8;    // [8]
    volatile int* dead = flags + 16;
    volatile uint32_t* tmem_at = reinterpret_cast<volatile uint32_t*>(flags + 17);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    sh_wait_before();
    sh_let_next();
    const int64_t total = sh_scan(a, L, scan);
    const int n_workers = sh_workers(L, total);
    if ((int)blockIdx.x >= n_workers) return;
    ShCursor cur;
    sh_seek(a, L, scan, n_workers, blockIdx.x, cur);
    if (cur.left <= 0) return;
    if (tid == 0) {
        *dead = 0;
        for (int i = 0; i < kTcRaw; ++i) {
            mbar_init(&bar[kRawKFull + i], 1);
            mbar_init(&bar[kRawVFull + i], 1);
            mbar_init(&bar[kRawKEmpty + i], 4);
            mbar_init(&bar[kRawVEmpty + i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar[kKFull + i], 4);
            mbar_init(&bar[kVFull + i], 4);
            mbar_init(&bar[kKEmpty + i], 1);
            mbar_init(&bar[kVEmpty + i], 1);
            mbar_init(&bar[kSFull + i], 1);
            mbar_init(&bar[kPFull + i], 4);
        }
        mbar_init(&bar[kQFull], 4);
        mbar_init(&bar[kPvDone], 1);
        mbar_init(&bar[kDrain], 1);
        fence_mbar_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(const_cast<uint32_t*>(tmem_at)))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_at;

    if (warp < 4) {
        // ---------------- softmax: row `rl` of the item's block ----------------
        const uint32_t lane_at = tmem + ((uint32_t)(32 * warp) << 16);
        const int rl = 32 * warp + lane;
        float sc = 0.0f, U = kShNone, l = 0.0f;
        bool begin = true, busy = false, valid = false, ok = true;
        for (int i = 0; cur.left > 0; ++i) {
            const int b = i & 1;
            if (begin) {
                const __half* src = rl < L.rows ? sh_query(a, L, cur, cur.blk * L.rows + rl, D) : nullptr;
                valid = src != nullptr;
                busy = __any_sync(0xffffffffu, valid);
                U = kShNone;
                l = 0.0f;
                if (busy) {
                    uint32_t x[D / 2];
                    if (!valid) {
#pragma unroll
                        for (int k = 0; k < D / 2; ++k) x[k] = 0;
                    } else if (a.q_aligned) {
#pragma unroll
                        for (int k = 0; k < D / 8; ++k) {
                            const uint4 v = reinterpret_cast<const uint4*>(src)[k];
                            x[4 * k] = v.x;
                            x[4 * k + 1] = v.y;
                            x[4 * k + 2] = v.z;
                            x[4 * k + 3] = v.w;
                        }
                    } else {
                        const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
                        for (int k = 0; k < D / 2; ++k) x[k] = s16[2 * k] | ((uint32_t)s16[2 * k + 1] << 16);
                    }
                    float mag = 0.0f;
#pragma unroll
                    for (int k = 0; k < D / 2; ++k) {
                        const float2 f = __half22float2(bits_h2(x[k]));
                        mag += fabsf(f.x) + fabsf(f.y);
                    }
                    const float mean = mag * (1.0f / D);
                    const __half h = __float2half_rn(mean);
                    const float hf = __half2float(h);
                    const float f = hf == 0.0f ? 1.0f : mean / hf;
                    sc = f * kShLog2e * rsqrtf((float)D);
                    const uint32_t hb = __half_as_ushort(h);
                    // sign part: pairs (i, i + 16) of each word
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        uint32_t r[16];
#pragma unroll
                        for (int p = 0; p < 16; ++p) {
                            const int d0 = 32 * w + p, d1 = d0 + 16;
                            const float f0 = d0 % 2 ? __high2float(bits_h2(x[d0 / 2])) : __low2float(bits_h2(x[d0 / 2]));
                            const float f1 = d1 % 2 ? __high2float(bits_h2(x[d1 / 2])) : __low2float(bits_h2(x[d1 / 2]));
                            r[p] = (hb | (f0 >= 0.0f ? 0u : 0x8000u)) | ((hb | (f1 >= 0.0f ? 0u : 0x8000u)) << 16);
                        }
                        tc_st16(lane_at + C::Q_COL + 16 * w, r);
                    }
                    if constexpr (COMP) {
                        const float g = (8.0f / 7.0f) / f;
#pragma unroll
                        for (int w = 0; w < NW; ++w) {
                            uint32_t r[16];
#pragma unroll
                            for (int p = 0; p < 16; ++p) {
                                const int d0 = sh_code_dim(D, 32 * w + 2 * p), d1 = sh_code_dim(D, 32 * w + 2 * p + 1);
                                const float f0 = d0 % 2 ? __high2float(bits_h2(x[d0 / 2])) : __low2float(bits_h2(x[d0 / 2]));
                                const float f1 = d1 % 2 ? __high2float(bits_h2(x[d1 / 2])) : __low2float(bits_h2(x[d1 / 2]));
                                r[p] = h2_bits(__floats2half2_rn(f0 * g, f1 * g));
                            }
                            tc_st16(lane_at + C::Q_COL + D / 2 + 16 * w, r);
                        }
                    }
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&bar[kQFull]);
            }
            ok = __all_sync(0xffffffffu, tc_wait(&bar[kSFull + b], (uint32_t)(i >> 1) & 1u, dead));
            if (!ok) break;
            tc_fence_after();
            if (busy) {
                const uint32_t s_at = lane_at + C::S_COL + 128 * b;
                const int kpos = (cur.x.tile0 + cur.tile) * kTcTile;
                const bool bad = kbad[i & 7] != 0;
                const int lo = bad ? kTcTile : max(0, cur.x.lo - kpos), hi = min(kTcTile, cur.x.hi - kpos);
                const bool masked = lo > 0 || hi < kTcTile;
                uint32_t v[32];
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tc_ld32(s_at + 32 * c, v);
                    tc_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (32 * c + k >= lo && 32 * c + k < hi) top = fmaxf(top, __uint_as_float(v[k]));
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) top = fmaxf(top, __uint_as_float(v[k]));
                    }
                }
                top *= sc;
                if (__any_sync(0xffffffffu, top - U > 15.0f)) {
                    const float U1 = top - U > 15.0f ? top - 8.0f : U, f = exp2f(U - U1);
                    U = U1;
                    l *= f;
                    if (!begin) {  // O holds the piece's tiles so far, once their products are through
                        ok = __all_sync(0xffffffffu, tc_wait(&bar[kPvDone], (uint32_t)(i - 1) & 1u, dead));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            tc_ld32(lane_at + C::O_COL + 32 * c, v);
                            tc_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                            tc_st32(lane_at + C::O_COL + 32 * c, v);
                        }
                        tc_wait_st();
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tc_ld32(s_at + 32 * c, v);
                    tc_wait_ld();
                    uint32_t p[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float e0 = exp2f(__uint_as_float(v[k]) * sc - U), e1 = exp2f(__uint_as_float(v[k + 1]) * sc - U);
                        if (masked) {
                            if (32 * c + k < lo || 32 * c + k >= hi) e0 = 0.0f;
                            if (32 * c + k + 1 < lo || 32 * c + k + 1 >= hi) e1 = 0.0f;
                        }
                        l += e0 + e1;
                        p[k / 2] = h2_bits(__floats2half2_rn(e0, e1));
                    }
                    tc_st16(s_at + 16 * c, p);
                }
                tc_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) tc_arrive(&bar[kPFull + b]);
            if (sh_piece_ends(cur)) {
                ok = __all_sync(0xffffffffu, tc_wait(&bar[kPvDone], (uint32_t)i & 1u, dead));
                if (!ok) break;
                tc_fence_after();
                if (busy) {
                    float* row = sh_record(a, L, cur, blockIdx.x, D) + rl * (D + 4);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t v[32];
                        tc_ld32(lane_at + C::O_COL + 32 * c, v);
                        tc_wait_ld();
                        if (valid) {
#pragma unroll
                            for (int k = 0; k < 32; k += 4)
                                *reinterpret_cast<uint4*>(row + 32 * c + k) = make_uint4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                        }
                    }
                    if (valid) *reinterpret_cast<float2*>(row + D) = make_float2(U, l);
                }
                tc_fence_before();
            }
            begin = sh_next(a, L, cur);
        }
    } else if (warp < 8) {
        // ---------------- unpack K: key `key` of each tile ----------------
        const int key = tid - 128;
        for (int i = 0; cur.left > 0; ++i) {
            const int rs_ = i % kTcRaw, b = i & 1;
            const uint8_t* raw = smem + C::RAWK_OFF + rs_ * C::RAW_B;
            bool ok = tc_wait(&bar[kRawKFull + rs_], (uint32_t)(i / kTcRaw) & 1u, dead);
            uint32_t sg[NW];
            uint4 nb[COMP ? NW : 1];
#pragma unroll
            for (int w = 0; w < NW; ++w) sg[w] = reinterpret_cast<const uint32_t*>(raw)[key * NW + w];
            const uint32_t bs = *reinterpret_cast<const uint16_t*>(raw + C::BS_OFF + 2 * key);
            uint32_t rs = 0;
            if constexpr (COMP) {
                rs = *reinterpret_cast<const uint16_t*>(raw + C::RS_OFF + 2 * key);
#pragma unroll
                for (int c = 0; c < NW; ++c)
                    nb[c] = *reinterpret_cast<const uint4*>(raw + C::SIGN_B + (key >> 3) * 4 * D + c * 128 + (key & 7) * 16);
            }
            __syncwarp();
            if (lane == 0) tc_arrive(&bar[kRawKEmpty + rs_]);
            if (i >= 2) ok = ok && tc_wait(&bar[kKEmpty + b], (uint32_t)((i >> 1) - 1) & 1u, dead);
            if (!__all_sync(0xffffffffu, ok)) break;
            uint8_t* op = smem + b * C::KOP_B + key * 128;
            const int sw = key & 7;
            const uint32_t flip = (bs | (bs << 16)) ^ 0x80008000u;
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int u = 4 * w + k;
                    sts128(op + (u >> 3) * (kTcTile * 128) + (((u & 7) ^ sw) << 4), tc_sign(sg[w], 4 * k, flip),
                           tc_sign(sg[w], 4 * k + 1, flip), tc_sign(sg[w], 4 * k + 2, flip), tc_sign(sg[w], 4 * k + 3, flip));
                }
            if constexpr (COMP) {
                const __half2 r8 = __hmul2(bits_h2(rs | (rs << 16)), bits_h2(0x30003000u));  // rs / 8
#pragma unroll
                for (int c = 0; c < NW; ++c) {
                    const uint32_t w4[4] = {nb[c].x, nb[c].y, nb[c].z, nb[c].w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int u = D / 8 + 4 * c + w;
                        uint32_t o[4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) o[t] = h2_bits(__hmul2(tc_code(w4[w], t), r8));
                        sts128(op + (u >> 3) * (kTcTile * 128) + (((u & 7) ^ sw) << 4), o[0], o[1], o[2], o[3]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc_arrive(&bar[kKFull + b]);
            sh_next(a, L, cur);
        }
    } else if (warp < 12) {
        // ---------------- unpack V ----------------
        const int key = tid - 256;
        for (int i = 0; cur.left > 0; ++i) {
            const int rs_ = i % kTcRaw, b = i % C::VST;
            const uint8_t* raw = smem + C::RAWV_OFF + rs_ * C::RAW_B;
            bool ok = tc_wait(&bar[kRawVFull + rs_], (uint32_t)(i / kTcRaw) & 1u, dead);
            uint32_t sg[NW];
            uint4 nb[COMP ? NW : 1];
#pragma unroll
            for (int w = 0; w < NW; ++w) sg[w] = reinterpret_cast<const uint32_t*>(raw)[key * NW + w];
            uint32_t bs = *reinterpret_cast<const uint16_t*>(raw + C::BS_OFF + 2 * key);
            uint32_t rs = 0;
            if constexpr (COMP) {
                rs = *reinterpret_cast<const uint16_t*>(raw + C::RS_OFF + 2 * key);
#pragma unroll
                for (int c = 0; c < NW; ++c)
                    nb[c] = *reinterpret_cast<const uint4*>(raw + C::SIGN_B + (key >> 3) * 4 * D + c * 128 + (key & 7) * 16);
            }
            // keys outside the prefix: P is 0 there, V has to be finite
            const int pos = (cur.x.tile0 + cur.tile) * kTcTile + key;
            if (vbad[i & 7] || pos < cur.x.lo || pos >= cur.x.hi) bs = rs = 0;
            __syncwarp();
            if (lane == 0) tc_arrive(&bar[kRawVEmpty + rs_]);
            if (i >= C::VST) ok = ok && tc_wait(&bar[kVEmpty + b], (uint32_t)(i / C::VST - 1) & 1u, dead);
            if (!__all_sync(0xffffffffu, ok)) break;
            uint8_t* op = smem + C::V_OFF + b * C::VOP_B + key * 128;
            const int sw = key & 7;
            const uint32_t flip = (bs | (bs << 16)) ^ 0x80008000u;
            const __half r7 = __float2half_rn(__half2float(__ushort_as_half((uint16_t)rs)) * (1.0f / 7.0f));
            const __half2 r72 = __half2half2(r7);
#pragma unroll
            for (int c = 0; c < NW; ++c) {
                uint32_t w4[4] = {0, 0, 0, 0};
                if constexpr (COMP) {
                    w4[0] = nb[c].x;
                    w4[1] = nb[c].y;
                    w4[2] = nb[c].z;
                    w4[3] = nb[c].w;
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    // nibble n of word w is bit 4n + first of sign word `word`
                    const int word = D == 128 ? w : D == 64 ? w % 2 : 4 * (c / 4) + w;
                    const int first = D == 128 ? c : D == 64 ? 2 * c + w / 2 : c % 4;
                    const int u = 4 * c + w;
                    uint32_t o[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t s = tc_sign(sg[word], 4 * t + first, flip);
                        o[t] = COMP ? h2_bits(__hfma2(tc_code(w4[w], t), r72, bits_h2(s))) : s;
                    }
                    sts128(op + (u >> 3) * (kTcTile * 128) + (((u & 7) ^ sw) << 4), o[0], o[1], o[2], o[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc_arrive(&bar[kVFull + b]);
            sh_next(a, L, cur);
        }
    } else if (warp == 12) {
        // ---------------- products ----------------
        if (lane == 0) {
            const uint32_t k0 = smem_u32(smem), v0 = smem_u32(smem + C::V_OFF);
            bool ok = true, pending = false, pv_first = true;
            auto values = [&](int j) {  // O (+)= P(j) V(j)
                ok = ok && tc_wait(&bar[kPFull + (j & 1)], (uint32_t)(j >> 1) & 1u, dead) &&
                     tc_wait(&bar[kVFull + j % C::VST], (uint32_t)(j / C::VST) & 1u, dead);
                if (!ok) return;
                tc_fence_after();
                const uint32_t at = v0 + (j % C::VST) * C::VOP_B;
#pragma unroll
                for (int k = 0; k < kTcTile / 16; ++k)
                    tc_mma(tmem + C::O_COL, tmem + C::S_COL + 128 * (j & 1) + 8 * k, tc_desc(at + 2048 * k, kTcTile * 128),
                           tc_idesc(D, true), !(pv_first && k == 0));
                tc_commit(&bar[kVEmpty + j % C::VST]);
                tc_commit(&bar[kPvDone]);
            };
            bool begin = true;
            int i = 0, items = 0;
            for (; ok && cur.left > 0; ++i) {
                const int b = i & 1;
                if (begin) {
                    if (pending) values(i - 1);  // the next item's queries come after the last one's results
                    pending = false;
                    ok = ok && tc_wait(&bar[kQFull], (uint32_t)items & 1u, dead);
                    ++items;
                }
                ok = ok && tc_wait(&bar[kKFull + b], (uint32_t)(i >> 1) & 1u, dead);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < C::KE / 16; ++k)
                    tc_mma(tmem + C::S_COL + 128 * b, tmem + C::Q_COL + 8 * k,
                           tc_desc(k0 + b * C::KOP_B + (k >> 2) * (kTcTile * 128) + (k & 3) * 32, 16), tc_idesc(kTcTile, false),
                           k > 0);
                tc_commit(&bar[kKEmpty + b]);
                tc_commit(&bar[kSFull + b]);
                if (pending) {
                    values(i - 1);
                    pv_first = false;
                }
                if (begin) pv_first = true;
                pending = true;
                begin = sh_next(a, L, cur);
            }
            if (pending) values(i - 1);
            if (!ok) raise_device_error(a.err, BC_DEVERR_TIMEOUT);
            tc_commit(&bar[kDrain]);
            for (uint32_t it = 0; it < kTcSpin; ++it)
                if (mbar_try_wait(&bar[kDrain], 0)) break;
        }
    } else {
        // ---------------- packed tiles of K (warp 13) or V (warp 14) ----------------
        if (lane == 0) {
            const bool is_v = warp == 14;
            const bc_kv_planes& P = is_v ? a.V : a.K;
            uint8_t* ring = smem + (is_v ? C::RAWV_OFF : C::RAWK_OFF);
            uint64_t* full = bar + (is_v ? kRawVFull : kRawKFull);
            uint64_t* empty = bar + (is_v ? kRawVEmpty : kRawKEmpty);
            volatile int* flag = is_v ? vbad : kbad;
            bool ok = true;
            int i = 0;
            for (; cur.left > 0; ++i) {
                const int s = i % kTcRaw;
                if (i >= kTcRaw) ok = tc_wait(&empty[s], (uint32_t)(i / kTcRaw - 1) & 1u, dead);
                if (!ok) break;
                const int pos = (cur.x.tile0 + cur.tile) * kTcTile;
                const int j = pos / a.pt.page_size;
                const int pg = __ldg(a.pt.pages + ((int64_t)sh_lead(a, L, cur) * a.n_kv + cur.h) * a.pt.max_pages + j);
                const bool here = pg >= 0 && pg < a.pt.n_pages;
                flag[i & 7] = !here;
                if (here) {
                    const int64_t row = (int64_t)pg * a.pt.page_size + (pos - j * a.pt.page_size);
                    uint8_t* dst = ring + s * C::RAW_B;
                    fence_proxy_async_smem();
                    mbar_arrive_expect_tx(&full[s], C::RAW_B);
                    bulk_g2s(dst, (const uint8_t*)P.sign + row * (D / 8), C::SIGN_B, &full[s]);
                    bulk_g2s(dst + C::BS_OFF, (const uint8_t*)P.bscale + row * 2, C::SC_B, &full[s]);
                    if constexpr (COMP) {
                        bulk_g2s(dst + C::SIGN_B, (const uint8_t*)P.nib + row * (D / 2), C::NIB_B, &full[s]);
                        bulk_g2s(dst + C::RS_OFF, (const uint8_t*)P.rscale + row * 2, C::SC_B, &full[s]);
                    }
                } else {
                    if (!is_v) raise_device_error(a.err, BC_DEVERR_PAGE);
                    tc_arrive(&full[s]);
                }
                sh_next(a, L, cur);
            }
            // copies in flight land before the block's memory is given back (bounded)
            for (int t = max(0, i - kTcRaw); t < i; ++t)
                for (uint32_t it = 0; it < kTcSpin; ++it)
                    if (mbar_try_wait(&full[t % kTcRaw], (uint32_t)(t / kTcRaw) & 1u)) break;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D, bool COMP>
int tc_run(const SharedArgs& a, const ShList& L, cudaStream_t st) {
    constexpr int smem = TcCfg<D, COMP>::SMEM_B;
    static_assert(smem <= 232448, "shared memory of one CTA");
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return BC_ERR_CUDA_BASE + (int)e;
    if (dev < 0 || dev >= 64) return BC_ERR_UNSUPPORTED;
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(k_shared_prefix<D, COMP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return BC_ERR_CUDA_BASE + (int)e;
        ready[dev] = true;
    }
    e = sh_launch(k_shared_prefix<D, COMP>, L.n_workers, kTcThreads, smem, st, a, L);
    return e == cudaSuccess ? BC_OK : BC_ERR_CUDA_BASE + (int)e;
}

}  // namespace

ShList sh_tc_list(int n_seqs, int n_groups, int group) {
    ShList L{};
    const int64_t rows = (int64_t)(n_seqs / n_groups) * group;
    L.n_pre = n_groups;
    L.pre_blocks = (int)((rows + 127) / 128);
    L.rows = (int)((rows + L.pre_blocks - 1) / L.pre_blocks);
    L.rows = (L.rows + 7) / 8 * 8;
    L.own_blocks = 1;
    L.tile = kTcTile;
    L.cost = kTcItemCost;
    return L;
}

int sh_tc_run(const SharedArgs& a, const ShList& L, int head_dim, bool compensated, cudaStream_t st) {
    if (head_dim == 128) return compensated ? tc_run<128, true>(a, L, st) : tc_run<128, false>(a, L, st);
    return compensated ? tc_run<64, true>(a, L, st) : tc_run<64, false>(a, L, st);
}

}  // namespace bc
