// What the kernels of bc_decode_attention_shared have in common: their arguments,
// the list of work and its even division, and the records of pieces.
#pragma once

#include "common.cuh"

namespace bc {

constexpr int kShThreads = 128;  // threads that take part in a list's sums
constexpr float kShLog2e = 1.4426950408889634f;
constexpr float kShNone = -1e30f;  // unit U of a row without keys

struct SharedArgs {
    const __half* q;
    bc_kv_planes K, V;
    bc_page_table pt;
    const int32_t* seq_lens;
    const int32_t* prefix_lens;  // null: no prefixes
    __half* out;
    unsigned int* err;
    int n_seqs, n_groups, per;  // per: sequences of a group
    int n_kv, group;
    bool q_aligned;  // q on a 16-byte boundary
};

// One kernel's list of work: entries [0, n_pre) are the groups' prefixes, the
// following n_own the sequences' own keys.  An item is one block of query rows of
// one kv head of an entry.
struct ShList {
    int n_pre, n_own;
    int pre_blocks, own_blocks;  // blocks of `rows` query rows of a prefix / of a sequence
    int shift, rows;             // keys of a tile: 2^shift; query rows of a block
    int copies;                  // rows of a record for each query row: the keys of a tile may be split among copies of it
    int cost;                    // an item's start and end, in tiles
    int n_workers;
    float* records;
};

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

// Entry e of a list.  A sequence shorter than its group's prefix takes no part in
// it (its rows there are not read) and attends all of its keys on its own.
struct ShEntry {
    int lo, hi;  // key positions
    int tile0, tiles;
    int blocks;
};
__device__ __forceinline__ ShEntry sh_entry(const SharedArgs& a, const ShList& L, int e) {
    ShEntry x;
    if (e < L.n_pre) {
        x.lo = 0;
        x.hi = sh_prefix(a, e);
        x.blocks = L.pre_blocks;
    } else {
        const int b = e - L.n_pre, prefix = sh_prefix(a, b / a.per);
        x.hi = sh_len(a, b);
        x.lo = x.hi < prefix ? 0 : prefix;
        x.blocks = L.own_blocks;
    }
    x.tile0 = x.lo >> L.shift;
    x.tiles = x.hi > x.lo ? ((x.hi - 1) >> L.shift) + 1 - x.tile0 : 0;
    return x;
}
__device__ __forceinline__ int sh_item_weight(const ShList& L, const ShEntry& x) { return x.tiles ? x.tiles + L.cost : 0; }
__device__ __forceinline__ int64_t sh_weight(const SharedArgs& a, const ShList& L, const ShEntry& x) {
    return (int64_t)sh_item_weight(L, x) * x.blocks * a.n_kv;
}
__host__ __device__ __forceinline__ int64_t sh_first_item(const ShList& L, int n_kv, int e) {
    return e < L.n_pre ? (int64_t)e * n_kv * L.pre_blocks
                       : ((int64_t)L.n_pre * L.pre_blocks + (int64_t)(e - L.n_pre) * L.own_blocks) * n_kv;
}

// Exclusive sums of the entries' weights over the CTA's first kShThreads threads
// (each a run of consecutive entries) in scan[0 .. kShThreads - 1]; the total
// behind them.
__device__ __forceinline__ int64_t sh_scan(const SharedArgs& a, const ShList& L, int64_t* scan) {
    const int n = L.n_pre + L.n_own, chunk = (n + kShThreads - 1) / kShThreads;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < kShThreads) {
        int64_t sum = 0;
        for (int e = threadIdx.x * chunk; e < min(n, ((int)threadIdx.x + 1) * chunk); ++e)
            sum += sh_weight(a, L, sh_entry(a, L, e));
        scan[threadIdx.x] = sum;
    }
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

// Worker w's stretch of the list: weights [sh_begin(w), sh_begin(w + 1)).  Within
// an item the first L.cost units stand for its start and end, the others for its
// tiles.  A piece's record is number item + worker: along the list every new
// piece raises one of the two.
__device__ __forceinline__ int sh_workers(const ShList& L, int64_t total) { return (int)min((int64_t)L.n_workers, total); }
// (Quotients in double precision: the products are below 2^53, and a quotient that
// is no whole number is further from one than the rounding of the division.)
__device__ __forceinline__ int64_t sh_begin(int64_t total, int n, int64_t w) {
    return (int64_t)((double)(total * w) / (double)n);
}
__device__ __forceinline__ int sh_worker_of(int64_t total, int n, int64_t at) {
    return (int)((double)((at + 1) * n + total - 1) / (double)total) - 1;
}
__device__ __forceinline__ int sh_tile_at(const ShList& L, int64_t at_in_item, int tiles) {
    return (int)max((int64_t)0, min((int64_t)tiles, at_in_item - L.cost));
}

// Position in a list; every thread keeps its own copy.
struct ShCursor {
    int e;
    ShEntry x;
    int h, blk, tile;  // tile: index within the item
    int64_t left;      // weight of the stretch from this tile on; <= 0 behind the last one
};
// The first tile of worker w's stretch.
__device__ __forceinline__ void sh_seek(const SharedArgs& a, const ShList& L, const int64_t* scan, int n_workers, int w,
                                        ShCursor& c) {
    const int64_t total = scan[kShThreads], w0 = sh_begin(total, n_workers, w);
    c.left = sh_begin(total, n_workers, w + 1) - w0;
    int run = 0;
#pragma unroll
    for (int step = kShThreads / 2; step; step >>= 1)
        if (scan[run + step] <= w0) run += step;
    const int n = L.n_pre + L.n_own, chunk = (n + kShThreads - 1) / kShThreads;
    int64_t at = w0 - scan[run];
    c.e = run * chunk;
    for (;; ++c.e) {
        c.x = sh_entry(a, L, c.e);
        const int64_t weight = sh_weight(a, L, c.x);
        if (at < weight) break;
        at -= weight;
    }
    const int one = sh_item_weight(L, c.x);
    const int it = (int)((double)at / (double)one);  // (exact: as sh_begin)
    const int in = (int)(at - (int64_t)it * one);
    c.h = it / c.x.blocks;
    c.blk = it - c.h * c.x.blocks;
    c.tile = sh_tile_at(L, in, c.x.tiles);
    c.left -= max(0, L.cost - in);
}
// Next tile of the stretch; true when it begins another item.  c.left tells whether there is one.
__device__ __forceinline__ bool sh_next(const SharedArgs& a, const ShList& L, ShCursor& c) {
    c.left -= 1;
    if (c.left <= 0 || ++c.tile < c.x.tiles) return false;
    c.left -= L.cost;
    if (c.left <= 0) return false;
    c.tile = 0;
    if (++c.blk < c.x.blocks) return true;
    c.blk = 0;
    if (++c.h < a.n_kv) return true;
    c.h = 0;
    do c.x = sh_entry(a, L, ++c.e);
    while (c.x.tiles == 0);
    return true;
}
// Tiles of the piece that begins at the cursor, and the step to the next one (a
// kernel's loop over tiles then has no list code in it).
__device__ __forceinline__ int sh_piece_tiles(const ShCursor& c) { return (int)min(c.left, (int64_t)(c.x.tiles - c.tile)); }
__device__ __forceinline__ void sh_next_piece(const SharedArgs& a, const ShList& L, ShCursor& c) {
    const int n = sh_piece_tiles(c) - 1;
    c.left -= n;
    c.tile += n;
    sh_next(a, L, c);
}
// The cursor's tile is the last of its piece.
__device__ __forceinline__ bool sh_piece_ends(const ShCursor& c) { return c.left <= 1 || c.tile + 1 == c.x.tiles; }
__device__ __forceinline__ float* sh_record(const SharedArgs& a, const ShList& L, const ShCursor& c, int worker, int d) {
    return L.records + (sh_first_item(L, a.n_kv, c.e) + (int64_t)c.h * c.x.blocks + c.blk + worker) * L.copies * L.rows * (d + 4);
}
__device__ __forceinline__ int sh_lead(const SharedArgs& a, const ShList& L, const ShCursor& c) {
    return c.e < L.n_pre ? c.e * a.per : c.e - L.n_pre;  // the sequence whose block table is read
}
// Query row r (0 ..) of the cursor's (entry, kv head): null past the last one.
__device__ __forceinline__ const __half* sh_query(const SharedArgs& a, const ShList& L, const ShCursor& c, int r, int d) {
    const int rows = c.e < L.n_pre ? a.per * a.group : a.group;
    if (r >= rows) return nullptr;
    return a.q + (((int64_t)(sh_lead(a, L, c) + r / a.group) * a.n_kv + c.h) * a.group + r % a.group) * d;
}
// Records hold the dims in the order of the packed codes: position n of word wi of
// chunk c (a pair n % 4, then n and n + 4) is element 8 (4 c + wi) + 2 (n % 4) + n / 4.
__host__ __device__ constexpr int sh_code_dim(int d, int at) {
    const int n = (at % 8) / 2 + 4 * (at % 2), u = at / 8;
    return nib_dim(d, u / 4, 4 * (u % 4) + n / 2, n % 2);
}
// Programmatic dependent launch: wait for the launch before this one / let the next one in.
__device__ __forceinline__ void sh_wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void sh_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launch that may begin while the one before it ends (its kernel waits by itself).
template <typename... Args>
inline cudaError_t sh_launch(void (*kernel)(Args...), int blocks, int threads, int smem, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace bc
