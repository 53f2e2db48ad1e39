// The prefix part of bc_decode_attention_shared when many query rows share a
// prefix: S = Q K^T and O += P V on the 5th-generation tensor cores.  sm_100a.
//
// An item is a block of up to 128 query rows of one kv head (M = 128, one row per
// tensor-memory lane) against a prefix, in tiles of 128 keys (N of the scores, K
// of the values).  A score needs two dots, sgn q . sgn k and q . n, with scales of
// the key's own, so K holds both parts side by side, scaled, and Q likewise:
//   K = [ bs sgn k | rs / 8 n ],  Q = [ h sgn q | q ] / 2^e,  h = fp16(7 / 8 mean|q|):
//   s = 8 / 7 2^e Q . K,  2^e <= mean|q| < 2^(e + 1), so that Q is exact but for h.
// (Without codes Q is sgn q, and s = mean|q| Q . K.)  V = bs sgn v + rs/7 n.
// The rows of K and V of each half tile (64 keys) are held in a unit of their own, 2^(E - 28)
// with E the exponent field of the half's largest scale, so that their largest elements
// lie at 2^13 .. 2^16: small scales become no fp16 subnormals (in which rs / 7 of 2e-5
// is 1% off), and bs + rs may pass the largest fp16.  K's unit goes back into the half's
// scores, V's into its P.  (One warp finds the units as tiles arrive; when each role found
// them for itself, 200000 keys before 32 rows took 219 us; 207 now, 199 without units.)
// A row of zeros has Q = 0 and a factor above 0, so that hidden keys' -inf stays -inf.
//
// Roles of the 28 warps of a CTA, one CTA per SM:
//   0-7    softmax: a thread owns a query row and half of every tile's keys (warps 0-3
//          keys 0-63, 4-7 the others).  Writes the row's Q (made by k_shared_queries)
//          into tensor memory, then per tile reads its scores, keeps U and l, writes P
//          (fp16, over the scores) and, when U moves, rescales O.  The two warps of a
//          row hand U on from one half tile to the next, so a half's maximum is known
//          before its weights are made and its values can go before the other's are
//          there (with maxima exchanged at every tile, one warp's waits were both's:
//          82 us instead of 78 in the case below).  Up to 32 rows stand four times
//          in the 128 lanes, each copy with a quarter of a half's keys; the copies are
//          joined with the pieces.
//   8-23   unpack: packed bytes -> fp16 operand rows in shared memory, two threads to a
//          key, 8-11 and 16-19 K, the others V.  K is K-major (128-byte swizzle, blocks
//          of 64 elements), V MN-major (dims contiguous).  The loops are rolled: fully
//          unrolled, waiting for instructions took more than everything else (13600
//          clocks a tile).
//   24     issues the products: Q (tensor memory) x K, P (tensor memory) x V.
//   25, 26 bring K's / V's packed tiles with 1-D bulk copies, three ahead.
//   27     finds the units of K's and V's half tiles.
// K's operand ring holds three half tiles (the sign part, the code part), V's two
// tiles.
//
// Keeping Q in tensor memory spares half of the score product's shared-memory
// reads.  Per tile 96 KB are written, 96 KB read by the tensor cores and 43 KB of
// packed bytes go in and out, 1900 clocks at 128 B each; the products take 1536, the
// exponentials of 128 rows 1024.  What bounds it: the chain from a tile's scores to the ones
// two tiles later in the same buffer, and the instructions of all roles, about 2500
// issue slots of a scheduler and tile (half of them unpacking; 55% of those there are),
// some 3300 clocks a tile; with few tiles, an item's start and end besides, about half
// of the time at 14 tiles a CTA.  128 sequences with 8192 keys before them, 32 / 8 heads of 128: 77 us with the batch's own keys, of
// which the products at the tensor cores' rate would take 15.  (Score products of 64
// keys, with four buffers, take as long each as those of 128: 229 us where these
// take 195, 32 rows before 200000 keys.)
//
// Scores are scaled so that P = 2^(s - U) times V's unit lies below 2^15, U rising when
// it would not, to 2^8 above the largest.  Sums are fp32.  The elements of K, V and P, h and
// V's rs / 7 are rounded to fp16, the widest type that the tensor cores take at this
// rate: with some channels four times the others, outputs are 5.0e-4 to 5.4e-4 off the exact
// ones, relative, of which their own fp16 rounding is 2.1e-4 and the five others 1.5e-4
// to 2.8e-4 each, none of them by itself worth the instructions that would spare it.
// Keys whose scales are below 2^-28 of their half tile's largest keep fewer bits.
// The rows kernel, which scales products in fp32 and rounds P alone, has 2.9e-4.
//
// A barrier tells odd phases from even ones, no more: whoever waits on one has to
// know that the phase before is over.  The value products have four in turn, one
// for each half tile, because the scores of tile i tell (the tensor cores work in
// order) that the values of tile i - 2 are through.  And since a row's two warps count
// tiles and pieces alike, whether they have rows in them or not (the last block of a kv
// head may fill fewer warps than the others), they arrive on each other's barriers for
// every one.  Those without rows do not wait there: that the phases before are over
// is known from the end of the values of a piece, which both warps have given their P.
#include "shared.cuh"
#include "shared_tc.h"

namespace bc {
namespace {

constexpr int kTcTile = 128;
constexpr int kTcThreads = 28 * 32;
constexpr int kTcUnpackWarps = 8;   // of K, and of V
constexpr int kTcRaw = 3;        // packed tiles ahead
constexpr int kTcItemCost = 2;   // an item's start and end, in tiles
constexpr uint64_t kTcPatience = 1000000000;  // ns before a wait gives up

template <int D, bool COMP>
struct TcCfg {
    static constexpr int KE = COMP ? 2 * D : D;              // elements of a K row
    static constexpr int PARTS = COMP ? 2 : 1;               // sign part, code part
    static constexpr int KOP_B = kTcTile * D * 2;            // one part of a K operand tile
    static constexpr int VOP_B = kTcTile * D * 2;
    static constexpr int KST = 3, VST = 2;                   // K operand parts, V operand tiles
    static constexpr int SIGN_B = kTcTile * D / 8;
    static constexpr int NIB_B = COMP ? kTcTile * D / 2 : 0;
    static constexpr int SC_B = kTcTile * 2;
    static constexpr int BS_OFF = SIGN_B + NIB_B;
    static constexpr int RS_OFF = BS_OFF + SC_B;
    static constexpr int RAW_B = SIGN_B + NIB_B + SC_B * (COMP ? 2 : 1);
    static constexpr int V_OFF = KST * KOP_B;
    static constexpr int RAWK_OFF = V_OFF + VST * VOP_B;
    static constexpr int RAWV_OFF = RAWK_OFF + kTcRaw * RAW_B;
    static constexpr int SCAN_OFF = (RAWV_OFF + kTcRaw * RAW_B + 15) / 16 * 16;
    static constexpr int XCH_OFF = SCAN_OFF;  // [2][128] units of the rows, [128] sums, once the list's sums are read
    static constexpr int BAR_OFF = SCAN_OFF + 512 * 4;
    static constexpr int FLAG_OFF = BAR_OFF + 52 * 8;
    static constexpr int UNIT_OFF = FLAG_OFF + 20 * 4;
    static constexpr int SMEM_B = UNIT_OFF + 4 * 8 * 8 + 1024;  // + alignment to the swizzle atom
    // tensor memory columns
    static constexpr int S_COL = 0, O_COL = 256, Q_COL = 256 + D;
    static_assert(Q_COL + KE / 2 <= 512, "tensor memory");
};

enum TcBar {
    kRawKFull = 0, kRawKEmpty = 3, kRawVFull = 6, kRawVEmpty = 9, kKFull = 12, kKEmpty = 15, kVFull = 18, kVEmpty = 20,
    kSFull = 22, kPFull = 26, kPvDone = 30, kQFull = 34, kDrain = 35, kPair = 36, kUnit = 40, kDone = 48, kScale = 49, kTcBars = 52
};

// ---- tcgen05 ---------------------------------------------------------------
// The issuing warp runs its loop with all lanes, and `one` picks the lane that
// issues: the addresses then live in uniform registers, which the instruction
// wants (from one lane's branch each product cost some 150 clocks to issue).
// A value that all lanes hold, in a uniform register.
__device__ __forceinline__ uint32_t tc_uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }
__device__ __forceinline__ uint32_t tc_elect() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 columns of 16 lanes: lane t gets columns 8 j + 2 (t % 4), + 1 of rows t / 4 (r[4 j], r[4 j + 1]) and
// t / 4 + 8, so that four lanes hold 32 consecutive bytes of a row.
__device__ __forceinline__ void tc_ld_rows(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
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
// Bounded in time; once one has given up (dead), all do, and the CTA winds down.
// The hint lets a waiting warp sleep until the phase ends: without it the polls of
// a dozen waiting warps were a third of all instructions.
__device__ __forceinline__ bool tc_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t tc_now() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
    if (tc_try_wait(bar, parity)) return true;
    const uint64_t limit = tc_now() + kTcPatience;
#pragma unroll 1
    while (!tc_try_wait(bar, parity)) {
        if (*dead) return false;
        if (tc_now() > limit) {
            *dead = 1;
            return false;
        }
    }
    return true;
}
// The last waits of a warp, for what it has set off itself.
__device__ __forceinline__ void tc_settle(uint64_t* bar, uint32_t parity, volatile int* dead) {
    const uint64_t limit = tc_now() + kTcPatience;
#pragma unroll 1
    while (!tc_try_wait(bar, parity)) {
        if (tc_now() > limit) {
            *dead = 1;
            return;
        }
    }
}
__device__ __forceinline__ void tc_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A warp's end: its use of tensor memory is over.
__device__ __forceinline__ void tc_leave(uint64_t* done) {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc_arrive(done);
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

__device__ __forceinline__ float2 tc_fma2(float2 x, float2 y, float2 z) {
    unsigned long long r;
    asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;"
        : "=l"(r)
        : "l"(*reinterpret_cast<unsigned long long*>(&x)), "l"(*reinterpret_cast<unsigned long long*>(&y)),
          "l"(*reinterpret_cast<unsigned long long*>(&z)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 tc_add2(float2 x, float2 y) {
    unsigned long long r;
    asm("add.rn.ftz.f32x2 %0, %1, %2;"
        : "=l"(r)
        : "l"(*reinterpret_cast<unsigned long long*>(&x)), "l"(*reinterpret_cast<unsigned long long*>(&y)));
    return *reinterpret_cast<float2*>(&r);
}

// Exponent field (0 .. 30) of the largest scale of a half tile's keys [lo, hi); bs: its packed scales.  A warp's call.
// (An infinite or NaN scale counts as 2^15.)
template <bool COMP>
__device__ __forceinline__ int tc_half_exp(const uint8_t* bs, int lo, int hi) {
    const int lane = threadIdx.x & 31, k = 2 * lane;
    uint32_t w = reinterpret_cast<const uint32_t*>(bs)[lane] & 0x7FFF7FFFu;
    if constexpr (COMP) w = __vmaxu2(w, reinterpret_cast<const uint32_t*>(bs + 2 * kTcTile)[lane] & 0x7FFF7FFFu);
    const uint32_t a = k >= lo && k < hi ? w & 0xFFFFu : 0, b = k + 1 >= lo && k + 1 < hi ? w >> 16 : 0;
    return min(30, (int)(__reduce_max_sync(0xffffffffu, max(a, b)) >> 10));
}
__device__ __forceinline__ float tc_pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ float half_at(const uint8_t* p) { return __half2float(*reinterpret_cast<const __half*>(p)); }

// The query rows as A operands, one warp a row: [h sgn q | q] / 2^e in the order of
// K's elements, and the scale of the row's scores in log2 units.  Ordered as the
// prefix kernel's lanes read them: by group and kv head, then 16-byte unit, then
// row.  A kernel of its own: a softmax thread that made its row itself ran some 800
// instructions once, at the pace of their fetch (12000 clocks a piece).
constexpr int kTcQueryWarps = 8;
template <int D, bool COMP>
__global__ void __launch_bounds__(32 * kTcQueryWarps) k_shared_queries(const SharedArgs a, uint32_t* __restrict__ ops,
                                                                       float* __restrict__ scales) {
    constexpr int WORDS = (COMP ? 2 : 1) * D / 2;
    sh_wait_before();
    sh_let_next();
    // (unsigned: the heads of all sequences are below 2^31)
    const unsigned head = blockIdx.x * kTcQueryWarps + (threadIdx.x >> 5), slot = head / (unsigned)a.group;
    const int lane = threadIdx.x & 31, b = (int)(slot / (unsigned)a.n_kv);
    if (b >= a.n_seqs) return;
    // query row r of (group of sequences, kv head) `item`, of `rows`
    const int rows = a.per * a.group, seq = b % a.per;
    const int64_t item = (int64_t)(b / a.per) * a.n_kv + (slot - (unsigned)b * a.n_kv);
    const int r = seq * a.group + (int)(head - slot * a.group);
    uint32_t* op = ops + item * rows * WORDS + 4 * r;
    const __half* x = a.q + (int64_t)head * D;
    float mag = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) mag += fabsf(__half2float(x[32 * k + lane]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mag += __shfl_xor_sync(0xffffffffu, mag, o);
    const float mean = mag * (1.0f / D);
    const int e = mean != 0.0f ? (__float_as_int(mean) >> 23 & 255) - 127 : 0;
    const float down = mean < INFINITY ? __int_as_float((127 - e) << 23) : NAN;
    if (lane == 0)
        scales[item * rows + r] =
            (COMP ? 8.0f / 7.0f * __int_as_float((127 + e) << 23) : mean != 0.0f ? mean : 1.0f) * kShLog2e * rsqrtf((float)D);
    const uint32_t hb = __half_as_ushort(__float2half_rn(COMP ? mean * down * 0.875f : mean < INFINITY ? (float)(mean != 0.0f) : NAN));
#pragma unroll
    for (int k = 0; k < D / 64; ++k) {
        const int c = 32 * k + lane, d0 = 32 * (c / 16) + c % 16;
        op[(int64_t)(c / 4) * rows * 4 + c % 4] = (hb | (__half2float(x[d0]) >= 0.0f ? 0u : 0x8000u)) |
                                                  ((hb | (__half2float(x[d0 + 16]) >= 0.0f ? 0u : 0x8000u)) << 16);
        if constexpr (COMP)
            op[(int64_t)(D / 8 + c / 4) * rows * 4 + c % 4] =
                h2_bits(__floats2half2_rn(__half2float(x[sh_code_dim(D, 2 * c)]) * down, __half2float(x[sh_code_dim(D, 2 * c + 1)]) * down));
    }
}

template <int D, bool COMP>
__global__ void __launch_bounds__(kTcThreads, 1) k_shared_prefix(const SharedArgs a, const ShList L, const uint32_t* __restrict__ ops,
                                                                    const float* __restrict__ scales) {
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
    // unit of K's half tiles [2][8] (2^(28 - e), its inverse), and of V's (2^(28 - e), e - 28), tile i % 8
    volatile float2* kunit = reinterpret_cast<volatile float2*>(smem + C::UNIT_OFF);
    volatile float2* vunit = kunit + 16;
    const int tid = threadIdx.x, warp = (int)tc_uniform(tid >> 5), lane = tid & 31;

    // the queries' kernel has waited for all that came before; only its own results are waited for below
    sh_let_next();
    const int64_t total = sh_scan(a, L, scan);
    const int n_workers = sh_workers(L, total);
    // A CTA without tiles waits too: with all prefixes empty nobody else would, and the end of this grid has to
    // tell that of the queries' kernel.
    if ((int)blockIdx.x >= n_workers) {
        sh_wait_before();
        return;
    }
    ShCursor cur;
    sh_seek(a, L, scan, n_workers, blockIdx.x, cur);
    if (cur.left <= 0) {
        sh_wait_before();
        return;
    }
    if (tid == 0) {
        *dead = 0;
        for (int i = 0; i < kTcRaw; ++i) {
            mbar_init(&bar[kRawKFull + i], 1);
            mbar_init(&bar[kRawVFull + i], 1);
            mbar_init(&bar[kScale + i], 1);
            mbar_init(&bar[kRawKEmpty + i], kTcUnpackWarps);
            mbar_init(&bar[kRawVEmpty + i], kTcUnpackWarps);
        }
        for (int i = 0; i < C::KST; ++i) {
            mbar_init(&bar[kKFull + i], kTcUnpackWarps);
            mbar_init(&bar[kKEmpty + i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar[kVFull + i], kTcUnpackWarps);
            mbar_init(&bar[kVEmpty + i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar[kSFull + i], 1);
            mbar_init(&bar[kPFull + i], 4);
            mbar_init(&bar[kPvDone + i], 1);
            mbar_init(&bar[kPair + i], 1);
        }
        mbar_init(&bar[kQFull], 8);
        for (int i = 0; i < 8; ++i) mbar_init(&bar[kUnit + i], 1);
        mbar_init(&bar[kDrain], 1);
        mbar_init(&bar[kDone], kTcThreads / 32 - 1);
        fence_mbar_init();
    }
    if (warp == 24) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(const_cast<uint32_t*>(tmem_at)))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tc_uniform(*tmem_at);

    // registers: 256 x 112 + 512 x 56 + 128 x 48 of the 896 x 72 launched
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        // ---------------- softmax: row `rl` of the item's block, keys 64 half .. of every tile ----------------
        const int half = warp >> 2, quad = warp & 3;
        const uint32_t lane_at = tmem + ((uint32_t)(32 * quad) << 16);
        // few rows: copies of them fill the 128 lanes, and each copy takes its share of a half tile's keys
        const int copies = L.copies, copy = copies > 1 ? quad : 0, rl = 32 * quad + lane - copy * (128 / copies);
        const int key0 = 64 / copies * copy;  // this copy's first key of a half tile
        float* xch = reinterpret_cast<float*>(smem + C::XCH_OFF) + 32 * quad + lane;  // [2][128] units, [128] sums
        float sc = 0.0f, U = kShNone, l = 0.0f;
        sh_wait_before();
        bool ok = true;
        // the row's other warp's unit behind half tile j (of this piece; that behind j - 2 has been seen)
        auto follow = [&](int j) {
            ok = __all_sync(0xffffffffu, tc_wait(&bar[kUnit + 2 * quad + (j & 1)], (uint32_t)(j >> 1) & 1u, dead));
            const float U1 = xch[128 * (j & 1)];
            l *= exp2f(U - U1);
            U = U1;
        };
        for (int i = 0, piece = 0; ok && cur.left > 0; sh_next_piece(a, L, cur), ++piece) {
            const int begin = i, end = i + sh_piece_tiles(cur);
            const int rows = a.per * a.group, r = cur.blk * L.rows + rl;
            const int64_t item = (int64_t)cur.e * a.n_kv + cur.h;
            const bool valid = rl < L.rows && r < rows, busy = __any_sync(0xffffffffu, valid);
            if (busy && half < C::PARTS) {
                const uint32_t* op = ops + (item * (C::KE / 2) + D / 2 * half) * rows + 4 * (valid ? r : 0);
#pragma unroll
                for (int k0 = 0; k0 < D / 2; k0 += 32) {
                    uint32_t x[32];
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const uint4 w = valid ? __ldcg(reinterpret_cast<const uint4*>(op + (int64_t)(k0 + k) * rows)) : make_uint4(0, 0, 0, 0);
                        x[k] = w.x;
                        x[k + 1] = w.y;
                        x[k + 2] = w.z;
                        x[k + 3] = w.w;
                    }
                    const uint32_t to = lane_at + C::Q_COL + D / 2 * half + k0;
                    tc_st16(to, *reinterpret_cast<uint32_t(*)[16]>(x));
                    tc_st16(to + 16, *reinterpret_cast<uint32_t(*)[16]>(x + 16));
                }
                tc_wait_st();
            }
            sc = valid ? __ldcg(scales + item * rows + r) : 1.0f;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) tc_arrive(&bar[kQFull]);
            U = kShNone;
            l = 0.0f;
#pragma unroll 1
            for (; i < end; ++i) {
                const int t = 2 * i + half;
                ok = __all_sync(0xffffffffu, tc_wait(&bar[kSFull + (i & 1)], (uint32_t)(i >> 1) & 1u, dead));
                if (!ok) break;
                tc_fence_after();
                if (busy) {
                    const uint32_t s_at = lane_at + C::S_COL + 64 * (t & 3);
                    const int first = (cur.x.tile0 + cur.tile + i - begin) * kTcTile + 64 * half + key0;
                    const int lo = kbad[i & 7] ? 64 : cur.x.lo - first, hi = cur.x.hi - first;
                    const float sk = sc * kunit[8 * half + (i & 7)].y, vup = vunit[8 * half + (i & 7)].x, ev = vunit[8 * half + (i & 7)].y;
                    uint32_t v[64];  // (with copies, 16 of them)
                    tc_ld16(s_at + key0, *reinterpret_cast<uint32_t(*)[16]>(v));
                    if (copies == 1) {
#pragma unroll
                        for (int c = 1; c < 4; ++c) tc_ld16(s_at + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(v + 16 * c));
                    }
                    tc_wait_ld();
                    if (lo > 0 || hi < 64) {  // keys outside the prefix
#pragma unroll
                        for (int k = 0; k < 64; ++k)
                            if (k < lo || k >= hi) v[k] = 0xFF800000u;
                    }
                    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 16; ++k) m[k & 3] = fmaxf(m[k & 3], __uint_as_float(v[k]));
                    if (copies == 1) {
#pragma unroll
                        for (int k = 16; k < 64; ++k) m[k & 3] = fmaxf(m[k & 3], __uint_as_float(v[k]));
                    }
                    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * sk + ev;
                    if (t > 2 * begin) {
                        follow(t - 1);
                        if (!ok) break;
                    }
                    if (__any_sync(0xffffffffu, top - U > 15.0f)) {
                        const float U1 = top - U > 15.0f ? top - 8.0f : U, f = exp2f(U - U1);
                        U = U1;
                        l *= f;
                        if (t > 2 * begin) {  // O holds the piece's keys so far, once their products are through
                            ok = __all_sync(0xffffffffu, tc_wait(&bar[kPvDone + ((t - 1) & 3)], (uint32_t)((t - 1) >> 2) & 1u, dead));
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 16; ++c) {
                                const uint32_t at = lane_at + C::O_COL + 16 * c;
                                uint32_t o[16];
                                tc_ld16(at, o);
                                tc_wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tc_st16(at, o);
                            }
                        }
                    }
                    xch[128 * half] = U;
                    __syncwarp();
                    if (lane == 0) tc_arrive(&bar[kUnit + 2 * quad + half]);
                    // P of key k: column k / 2 of the half tile's, over scores that this warp has read
                    float2 sum = make_float2(0.0f, 0.0f);
                    const float2 sc2 = make_float2(sk, sk), U2 = make_float2(ev - U, ev - U);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c > 0 && copies > 1) continue;
                        uint32_t p[8];
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            float2 e = tc_fma2(make_float2(__uint_as_float(v[16 * c + k]), __uint_as_float(v[16 * c + k + 1])),
                                               sc2, U2);
                            e.x = exp2f(e.x);
                            e.y = exp2f(e.y);
                            sum = tc_add2(sum, e);
                            p[k / 2] = h2_bits(__floats2half2_rn(e.x, e.y));
                        }
                        tc_st8(s_at + (key0 >> 1) + 8 * c, p);
                    }
                    if (copies > 1) {  // the other copies' keys: P is 0
                        const uint32_t z[8] = {};
#pragma unroll 1
                        for (int c = 0; c < 4; ++c)
                            if (c != copy) tc_st8(s_at + 8 * c, z);
                    }
                    l += (sum.x + sum.y) * vup;
                    tc_wait_st();
                } else if (lane == 0) {
                    tc_arrive(&bar[kUnit + 2 * quad + half]);  // (kUnit and kPair count every tile and piece)
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&bar[kPFull + (t & 3)]);
            }
            if (!ok) break;
            if (busy) {  // the row's sum: both warps', in the unit of the piece's last keys, half 1's
                if (half == 0) {
                    follow(2 * end - 1);
                    if (!ok) break;
                    xch[256] = l;
                    __syncwarp();
                    if (lane == 0) tc_arrive(&bar[kPair + quad]);
                } else {
                    ok = __all_sync(0xffffffffu, tc_wait(&bar[kPair + quad], (uint32_t)piece & 1u, dead));
                    if (!ok) break;
                    l += xch[256];
                }
            } else if (half == 0 && lane == 0) {
                tc_arrive(&bar[kPair + quad]);
            }
            // (the last half tile but one first: its end tells that the phase before the last one's is over)
            for (int j = 2 * end - 2; ok && j < 2 * end; ++j)
                ok = __all_sync(0xffffffffu, tc_wait(&bar[kPvDone + (j & 3)], (uint32_t)(j >> 2) & 1u, dead));
            if (!ok) break;
            tc_fence_after();
            if (busy) {
                float* row = sh_record(a, L, cur, blockIdx.x, D) + (copy * L.rows + rl) * (D + 4);
                const unsigned live = __ballot_sync(0xffffffffu, valid);
                // 64 columns at a time (all of them at head_dim 64: one warp each half of the rows)
#pragma unroll 1
                for (int s16 = D == 64 ? half : 0; s16 < (D == 64 ? half + 1 : 2); ++s16) {
                    uint32_t v[32];
                    const int col = D == 64 ? 0 : 64 * half;
                    tc_ld_rows(lane_at + ((uint32_t)(16 * s16) << 16) + C::O_COL + col, v);
                    tc_wait_ld();
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int at = 16 * s16 + 8 * y + (lane >> 2);  // the row's lane
                        float* to = row + (at - lane) * (D + 4) + col + 2 * (lane & 3);
                        if (live >> at & 1) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                *reinterpret_cast<uint2*>(to + 8 * j) = make_uint2(v[4 * j + 2 * y], v[4 * j + 2 * y + 1]);
                        }
                    }
                }
                if (valid && half == 1) *reinterpret_cast<float2*>(row + D) = make_float2(U, l);
            }
            tc_fence_before();
        }
        tc_leave(&bar[kDone]);
        return;
    }
    if (warp < 24) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        const int part = (warp - 8) >> 3, key = 32 * (warp & 3) + lane, sw = key & 7;
        int i = 0;
        bool ok = true;
        if (!(warp & 4)) {
            // ---------------- unpack K: words (and chunks) NW / 2 part .. of key `key` ----------------
            int slot = 0;
            uint32_t round = 0;  // of the operand ring
            auto next = [&]() {
                if (++slot == C::KST) {
                    slot = 0;
                    ++round;
                }
            };
            for (; ok && cur.left > 0; sh_next_piece(a, L, cur))
#pragma unroll 1
                for (const int end = i + sh_piece_tiles(cur); i < end; ++i) {
                    const int rs_ = i % kTcRaw;
                    const uint8_t* raw = smem + C::RAWK_OFF + rs_ * C::RAW_B;
                    ok = tc_wait(&bar[kScale + rs_], (uint32_t)(i / kTcRaw) & 1u, dead);
                    if (round) ok = ok && tc_wait(&bar[kKEmpty + slot], (round - 1) & 1u, dead);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    uint8_t* op = smem + slot * C::KOP_B + key * 128;
                    const float up = kunit[8 * (key >> 6) + (i & 7)].x;
                    const uint32_t flip = h2_bits(__float2half2_rn(half_at(raw + C::BS_OFF + 2 * key) * up)) ^ 0x80008000u;
#pragma unroll 1
                    for (int w = part * (NW / 2); w < (part + 1) * (NW / 2); ++w) {
                        const uint32_t sg = reinterpret_cast<const uint32_t*>(raw)[key * NW + w];
                        uint8_t* to = op + (w >> 1) * (kTcTile * 128);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            sts128(to + (((4 * (w & 1) + k) ^ sw) << 4), tc_sign(sg, 4 * k, flip), tc_sign(sg, 4 * k + 1, flip),
                                   tc_sign(sg, 4 * k + 2, flip), tc_sign(sg, 4 * k + 3, flip));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc_arrive(&bar[kKFull + slot]);
                    next();
                    if constexpr (COMP) {
                        if (round) ok = tc_wait(&bar[kKEmpty + slot], (round - 1) & 1u, dead);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        op = smem + slot * C::KOP_B + key * 128;
                        const __half2 r8 = __float2half2_rn(half_at(raw + C::RS_OFF + 2 * key) * (up * 0.125f));
#pragma unroll 1
                        for (int c = part * (NW / 2); c < (part + 1) * (NW / 2); ++c) {
                            const uint4 nb = *reinterpret_cast<const uint4*>(raw + C::SIGN_B + (key >> 3) * 4 * D + c * 128 + (key & 7) * 16);
                            const uint32_t w4[4] = {nb.x, nb.y, nb.z, nb.w};
                            uint8_t* to = op + (c >> 1) * (kTcTile * 128);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t o[4];
#pragma unroll
                                for (int t = 0; t < 4; ++t) o[t] = h2_bits(__hmul2(tc_code(w4[j], t), r8));
                                sts128(to + (((4 * (c & 1) + j) ^ sw) << 4), o[0], o[1], o[2], o[3]);
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) tc_arrive(&bar[kKFull + slot]);
                        next();
                    }
                    if (lane == 0) tc_arrive(&bar[kRawKEmpty + rs_]);
                }
        } else {
            // ---------------- unpack V: chunks NW / 2 part .. ----------------
            for (; ok && cur.left > 0; sh_next_piece(a, L, cur)) {
                int pos = (cur.x.tile0 + cur.tile) * kTcTile + key;
#pragma unroll 1
                for (const int end = i + sh_piece_tiles(cur); i < end; ++i, pos += kTcTile) {
                    const int rs_ = i % kTcRaw, b = i % C::VST;
                    const uint8_t* raw = smem + C::RAWV_OFF + rs_ * C::RAW_B;
                    ok = tc_wait(&bar[kScale + rs_], (uint32_t)(i / kTcRaw) & 1u, dead);
                    if (i >= C::VST) ok = ok && tc_wait(&bar[kVEmpty + b], (uint32_t)(i / C::VST - 1) & 1u, dead);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const float up = vunit[8 * (key >> 6) + (i & 7)].x;
                    float bs = half_at(raw + C::BS_OFF + 2 * key) * up, rs = COMP ? half_at(raw + C::RS_OFF + 2 * key) * (up * (1.0f / 7.0f)) : 0.0f;
                    // keys outside the prefix: P is 0 there, V has to be finite
                    if (vbad[i & 7] || pos < cur.x.lo || pos >= cur.x.hi) bs = rs = 0.0f;
                    uint8_t* op = smem + C::V_OFF + b * C::VOP_B + key * 128;
                    const uint32_t flip = h2_bits(__float2half2_rn(bs)) ^ 0x80008000u;
                    const __half2 r7 = __float2half2_rn(rs);
                    // chunk c: units 4c .. 4c + 3.  Nibble n of its word w is bit 4n + first of a sign
                    // word: word w, first c (head_dim 128); word w % 2, first 2c + w / 2 (64)
                    uint32_t sgw[NW];
                    if constexpr (D == 128) {
                        const uint4 x = *reinterpret_cast<const uint4*>(raw + key * 16);
                        sgw[0] = x.x;
                        sgw[1] = x.y;
                        sgw[2] = x.z;
                        sgw[3] = x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(raw + key * 8);
                        sgw[0] = x.x;
                        sgw[1] = x.y;
                    }
#pragma unroll 1
                    for (int c = part * (NW / 2); c < (part + 1) * (NW / 2); ++c) {
                        uint32_t w4[4] = {0, 0, 0, 0};
                        if constexpr (COMP) {
                            const uint4 nb = *reinterpret_cast<const uint4*>(raw + C::SIGN_B + (key >> 3) * 4 * D + c * 128 + (key & 7) * 16);
                            w4[0] = nb.x;
                            w4[1] = nb.y;
                            w4[2] = nb.z;
                            w4[3] = nb.w;
                        }
                        uint8_t* to = op + (c >> 1) * (kTcTile * 128);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t sg = D == 128 ? sgw[w % NW] >> c : sgw[w % 2] >> (2 * c + w / 2);
                            uint32_t o[4];
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const uint32_t x = tc_sign(sg, 4 * t, flip);
                                o[t] = COMP ? h2_bits(__hfma2(tc_code(w4[w], t), r7, bits_h2(x))) : x;
                            }
                            sts128(to + (((4 * (c & 1) + w) ^ sw) << 4), o[0], o[1], o[2], o[3]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tc_arrive(&bar[kVFull + b]);
                        tc_arrive(&bar[kRawVEmpty + rs_]);
                    }
                }
            }
        }
        tc_leave(&bar[kDone]);
        return;
    }
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 24) {
        // ---------------- products ----------------
        {
            const uint32_t one = tc_elect();
            const uint64_t kd = tc_desc(smem_u32(smem), 16), vd = tc_desc(smem_u32(smem + C::V_OFF), kTcTile * 128);
            bool ok = true;
            auto values = [&](int t, bool first) {  // O (+)= P V of half tile t
                const int j = t >> 1, h = t & 1;
                ok = __all_sync(0xffffffffu, ok && tc_wait(&bar[kPFull + (t & 3)], (uint32_t)(t >> 2) & 1u, dead) &&
                                                 (h || tc_wait(&bar[kVFull + j % C::VST], (uint32_t)(j / C::VST) & 1u, dead)));
                if (!ok) return;
                tc_fence_after();
                const uint64_t at = vd + (j % C::VST) * (C::VOP_B >> 4) + (2048 >> 4) * 4 * h;
                const uint32_t p = tmem + C::S_COL + 64 * (t & 3);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    tc_mma(tmem + C::O_COL, p + 8 * k, at + (2048 >> 4) * k, tc_idesc(D, true), !first || k > 0, one);
                if (h) tc_commit(&bar[kVEmpty + j % C::VST], one);
                tc_commit(&bar[kPvDone + (t & 3)], one);
            };
            int i = 0, slot = 0;
            uint32_t round = 0;
            for (int items = 0; __all_sync(0xffffffffu, ok && cur.left > 0); ++items, sh_next_piece(a, L, cur)) {
                const int from = i, end = i + (int)tc_uniform(sh_piece_tiles(cur));
                ok = __all_sync(0xffffffffu, tc_wait(&bar[kQFull], (uint32_t)items & 1u, dead));
                // the scores of a tile go before the values of the one before it; a piece's last values
                // before the next one's scores, whose queries are there only then
#pragma unroll 1
                for (; ok && i <= end; ++i) {
                    if (i < end) {
                        const int b = i & 1;
#pragma unroll 1
                        for (int part = 0; ok && part < C::PARTS; ++part) {
                            ok = __all_sync(0xffffffffu, tc_wait(&bar[kKFull + slot], round & 1u, dead));
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t at = kd + slot * (C::KOP_B >> 4);
                            const uint32_t qat = tmem + C::Q_COL + D / 2 * part;
#pragma unroll
                            for (int k = 0; k < D / 16; ++k)
                                tc_mma(tmem + C::S_COL + 128 * b, qat + 8 * k, at + 2 * k + (k >> 2) * ((kTcTile * 128 >> 4) - 8),
                                       tc_idesc(kTcTile, false), part + k > 0, one);
                            tc_commit(&bar[kKEmpty + slot], one);
                            if (++slot == C::KST) {
                                slot = 0;
                                ++round;
                            }
                        }
                        if (!ok) break;
                        tc_commit(&bar[kSFull + b], one);
                    }
                    if (i > from) {
                        values(2 * i - 2, i - 1 == from);
                        values(2 * i - 1, false);
                    }
                }
                i = end;
            }
            tc_commit(&bar[kDrain], one);
            tc_settle(&bar[kDrain], 0, dead);
        }
        __syncwarp();
        // the tensor memory goes back once all warps are through with it (bounded, as every wait)
        tc_settle(&bar[kDone], 0, dead);
        __syncwarp();
        if (*dead && lane == 0) raise_device_error(a.err, BC_DEVERR_TIMEOUT);
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        return;
    }
    if (warp == 25 || warp == 26) {
        // ---------------- packed tiles of K (warp 25) or V (warp 26) ----------------
        if (lane == 0) {
            const bool is_v = warp == 26;
            const bc_kv_planes& P = is_v ? a.V : a.K;
            uint8_t* ring = smem + (is_v ? C::RAWV_OFF : C::RAWK_OFF);
            uint64_t* full = bar + (is_v ? kRawVFull : kRawKFull);
            uint64_t* empty = bar + (is_v ? kRawVEmpty : kRawKEmpty);
            volatile int* flag = is_v ? vbad : kbad;
            bool ok = true;
            int i = 0;
            for (; ok && cur.left > 0; sh_next_piece(a, L, cur)) {
                const int pos = (cur.x.tile0 + cur.tile) * kTcTile, j = pos / a.pt.page_size;
                const int32_t* page = a.pt.pages + ((int64_t)sh_lead(a, L, cur) * a.n_kv + cur.h) * a.pt.max_pages + j;
                int in_page = pos - j * a.pt.page_size, pg = __ldg(page);
#pragma unroll 1
                for (const int end = i + sh_piece_tiles(cur); i < end; ++i) {
                    const int s = i % kTcRaw;
                    if (i >= kTcRaw) ok = tc_wait(&empty[s], (uint32_t)(i / kTcRaw - 1) & 1u, dead);
                    if (!ok) break;
                    const bool here = pg >= 0 && pg < a.pt.n_pages;
                    flag[i & 7] = !here;
                    if (here) {
                        const int64_t row = (int64_t)pg * a.pt.page_size + in_page;
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
                    in_page += kTcTile;
                    if (in_page == a.pt.page_size && i + 1 < end) {
                        in_page = 0;
                        pg = __ldg(++page);
                    }
                }
            }
            // copies in flight land before the block's memory is given back (bounded)
            for (int t = max(0, i - kTcRaw); t < i; ++t)
                tc_settle(&full[t % kTcRaw], (uint32_t)(t / kTcRaw) & 1u, dead);
        }
    }
    if (warp == 27) {
        // ---------------- units of the half tiles ----------------
        bool ok = true;
        int i = 0;
        for (; ok && cur.left > 0; sh_next_piece(a, L, cur)) {
            int at0 = (cur.x.tile0 + cur.tile) * kTcTile;
#pragma unroll 1
            for (const int end = i + sh_piece_tiles(cur); i < end; ++i, at0 += kTcTile) {
                const int s = i % kTcRaw;
                ok = tc_wait(&bar[kRawKFull + s], (uint32_t)(i / kTcRaw) & 1u, dead) &&
                     tc_wait(&bar[kRawVFull + s], (uint32_t)(i / kTcRaw) & 1u, dead);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint8_t *k = smem + C::RAWK_OFF + s * C::RAW_B + C::BS_OFF, *v = smem + C::RAWV_OFF + s * C::RAW_B + C::BS_OFF;
                const int lo = cur.x.lo - at0, khi = kbad[i & 7] ? 0 : cur.x.hi - at0, vhi = vbad[i & 7] ? 0 : cur.x.hi - at0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int ke = tc_half_exp<COMP>(k + 128 * h, lo - 64 * h, khi - 64 * h);
                    const int ve = tc_half_exp<COMP>(v + 128 * h, lo - 64 * h, vhi - 64 * h);
                    if (lane == 0) {
                        volatile float2 &ku = kunit[8 * h + (i & 7)], &vu = vunit[8 * h + (i & 7)];
                        ku.x = tc_pow2(28 - ke);
                        ku.y = tc_pow2(ke - 28);
                        vu.x = tc_pow2(28 - ve);
                        vu.y = (float)(ve - 28);
                    }
                }
                __syncwarp();
                if (lane == 0) tc_arrive(&bar[kScale + s]);
            }
        }
    }
    tc_leave(&bar[kDone]);
}

template <int D, bool COMP>
int tc_run(const SharedArgs& a, const ShList& L, void* scratch, cudaStream_t st) {
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
    const int64_t rows = (int64_t)a.n_seqs * a.n_kv * a.group;
    uint32_t* ops = (uint32_t*)scratch;
    float* scales = (float*)(ops + rows * (TcCfg<D, COMP>::KE / 2));
    e = sh_launch(k_shared_queries<D, COMP>, (int)((rows + kTcQueryWarps - 1) / kTcQueryWarps), 32 * kTcQueryWarps, 0, st,
                  a, ops, scales);
    if (e == cudaSuccess)
        e = sh_launch(k_shared_prefix<D, COMP>, L.n_workers, kTcThreads, smem, st, a, L, (const uint32_t*)ops,
                      (const float*)scales);
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
    // Up to 32 rows: four copies of the rows, each with a quarter of the keys, so that all softmax lanes work
    // (32 rows: 206 us at 200000 keys, 215 with one copy; 60.7 and 58.0 at 32768).  Two copies of 33 to 64 rows
    // cost more than they spare.
    L.copies = L.rows <= 32 ? 4 : 1;
    L.own_blocks = 1;
    L.shift = 7;
    L.cost = kTcItemCost;
    return L;
}

size_t sh_tc_scratch(int64_t rows, int head_dim) { return (size_t)rows * (4 * head_dim + 16); }

int sh_tc_run(const SharedArgs& a, const ShList& L, void* scratch, int head_dim, bool compensated, cudaStream_t st) {
    if (head_dim == 128) return compensated ? tc_run<128, true>(a, L, scratch, st) : tc_run<128, false>(a, L, scratch, st);
    return compensated ? tc_run<64, true>(a, L, scratch, st) : tc_run<64, false>(a, L, scratch, st);
}

}  // namespace bc
