// What the attention kernels over whole requests share (span_attention.cu, span_attention_tcgen05.cu): which rows see which keys,
// how the work is cut among the blocks, and where partial results meet.
//
// A request (a span) brings `len` rows behind `pos` keys that it holds already; all of their keys and values are in the cache, at
// the places 0 .. pos + len - 1 of its block table.  A row sees the `pos` keys and, of the keys of the rows it comes with,
//   tree     those that its mask names (bit j of its words: the key of row j of its request), or
//   causal   those up to its own.
// The G query heads of a kv head read the same keys, so the rows of a job are (row, head of the group) pairs, G to a row: a job is
// so many rows of one request and one kv head, over all key tiles that they see.  All jobs' tiles, one job after the other, make one
// line that is cut into equal lengths, one a block, whatever the lengths of the requests are: no block waits for a longer one.
// A job that a cut falls into leaves partial results (O, m, l), which a second kernel joins in the order of the blocks, so the
// result does not depend on which block is first.  (The block that leaves the last part could join them all: built, and slower. A
// trip to what other multiprocessors wrote takes 0.6 us, and one block has too few of them on their way: 8 nodes of one request
// 33 us instead of 18.)  Everything is worked out on the device: a captured graph serves other lengths.
#pragma once
#include "common.cuh"
#include "shared_memory.h"

constexpr int LLB_SPAN_BLOCKS = 512;          // blocks of a kernel at most
constexpr int LLB_SPAN_TC_LEAST = 2;          // tiles a block of the tensor-core kernel has at least: one for each of its groups
// What beginning and ending a job costs a block, in tiles: every job is so much longer in the line, or blocks with several short jobs would be the
// last ones (tensor cores, 27 trees of up to 26 rows behind 65 to 4,001 keys, 12/2 heads of 128: 45 us with nothing, 39 with one tile, 33 with 3
// or 5; 64 trees behind 30 to 300 keys, 28/4 heads: 38.5, 38, 37 with 3, 41 with 5.  CUDA cores, 5 trees of 64 rows: 51 with nothing, 48 with
// one, 53 with 3).
constexpr int LLB_SPAN_TC_EXTRA = 3, LLB_SPAN_EXTRA = 1;

struct LlbSpanArgs {
    const int* span_row;             // [S]
    const int* span_len;
    const int* span_pos;
    const int* table;                // [S, max_pages]
    int S, T, max_pages, page_size, max_len, num_slots;
    int page_shift;                  // log2 of the page size, or -1
    int Hq, Hkv, hd, group;
    const unsigned long long* mask;  // tree: [T, words]; null: causal
    int words;
    float scale_log2e;               // scores are kept in base-2 units
    const void* q;                   // [T, Hq, hd], keys [num_slots, Hkv, hd]
    const void* k;
    void* out;                       // [T, Hq, hd]
    float* lse;                      // [T, Hq] or null (causal rows): log2 of the sum of 2^score
    float* scores;                   // [score_tiles, group, keys a tile] or null: the scores of requests of one row, tile by tile of the line
    int score_tiles;                 // as many as the keys of the cache fill (tables that name pages outside the cache may make more)
    const float* mass_in;            // [Hkv, num_slots] or null: zeros
    float* mass;                     // [Hkv, num_slots]
    float* part_o;                   // [2 * blocks, ceil(hd / 4), rows, 4]: what a block has of a job that began before it (0) and goes on after
                                     // it (1); four dimensions of neighbouring rows side by side, as the threads that write and join them have them
    float* part_ml;                  // [2 * blocks, rows, 2]
    int* open;                       // [blocks, 4]: the job that begins in a block and goes on after it, see LlbOpen
    int extra;                       // what a job takes of the line besides its tiles
    int nodes;                       // rows of a request that a job holds at most
    int rows;                        // nodes * group, rounded up: (row, head) pairs of a job in the partial results
};

struct LlbSpan {
    int row, len, pos;
};
// What request s brings, held to what its arguments and the block table have room for.
__device__ __forceinline__ LlbSpan llb_span(const LlbSpanArgs& a, int s) {
    LlbSpan z;
    z.row = a.span_row[s];
    z.pos = max(a.span_pos[s], 0);
    z.len = min(min(a.span_len[s], a.max_len), min(a.T - z.row, a.max_pages * a.page_size - z.pos));
    if (z.row < 0 || z.len < 0) z.len = 0;
    return z;
}
// How many keys the rows up to `upto` (of the request) see between them.
__device__ __forceinline__ int llb_span_keys(const LlbSpanArgs& a, const LlbSpan& z, int upto) {
    return z.pos + (a.mask ? z.len : min(z.len, upto));
}
// The cache row of a key, or -1 for a page that is none of the cache's: such a key reads as zeros.
__device__ __forceinline__ int llb_span_slot(const LlbSpanArgs& a, int s, int key) {
    const int page_of = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
    const int page = a.table[(size_t)s * a.max_pages + page_of];
    const long long slot = (long long)page * a.page_size + (key - page_of * a.page_size);
    return page >= 0 && slot < a.num_slots ? (int)slot : -1;
}

// Two floats in a 64-bit register: an instruction for both.
__device__ __forceinline__ unsigned long long llb_pack2(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void llb_unpack2(unsigned long long v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ unsigned long long llb_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long llb_add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// A job and its tiles' place in the line of all tiles: begin .. begin + tiles - 1, then what it costs besides (no tile, and nothing to do for
// a block whose piece begins there).
struct LlbJob {
    LlbSpan z;
    int s, first, kvh;       // first: its first row in its request
    int keys, tiles, begin;  // begin: of its first tile in the line
    __device__ __forceinline__ void measure(const LlbSpanArgs& a, int tile) {
        keys = llb_span_keys(a, z, first + a.nodes);
        tiles = (keys + tile - 1) / tile;
    }
    __device__ __forceinline__ int count(const LlbSpanArgs& a) const { return min(a.nodes, z.len - first); }
    // the next job of the line (there is one)
    __device__ __forceinline__ void next(const LlbSpanArgs& a, int tile) {
        begin += tiles + a.extra;
        if (++kvh < a.Hkv) return;
        kvh = 0;
        first += a.nodes;
#pragma unroll 1
        while (first >= z.len) {
            ++s;
            z = llb_span(a, s);
            first = 0;
        }
        measure(a, tile);
    }
};
// A block's piece of the line: tiles [t0, t1), the job that t0 lies in; `blocks` of the grid have a piece.
struct LlbPiece {
    int t0, t1, total, blocks;
    LlbJob job;
    // The first total % blocks pieces are a tile longer than the others.
    __device__ __forceinline__ int start(int block) const { return block * (total / blocks) + min(block, total % blocks); }
    // Which block has tile t of the line.
    __device__ __forceinline__ int owner(int t) const {
        const int each = total / blocks, longer = total % blocks, head = longer * (each + 1);
        return t < head ? t / (each + 1) : longer + (t - head) / each;
    }
};
__device__ __forceinline__ int llb_span_tiles(const LlbSpanArgs& a, const LlbSpan& z, int tile) {
    int n = 0;
    if (z.len > 0 && a.mask) n = (z.len + a.nodes - 1) / a.nodes * ((z.pos + z.len + tile - 1) / tile + a.extra);
    else
#pragma unroll 1
        for (int c = 0; c < z.len; c += a.nodes) n += (llb_span_keys(a, z, c + a.nodes) + tile - 1) / tile + a.extra;
    return n * a.Hkv;
}
// By one whole warp; every lane gets the answer.  A block has `least` tiles or more where there are enough.
__device__ __forceinline__ LlbPiece llb_piece(const LlbSpanArgs& a, int tile, int block, int grid, int least, int lane) {
    LlbPiece p;
    LlbSpan z = {0, 0, 0};
    int mine = 0;
    p.total = 0;
#pragma unroll 1
    for (int base = 0; base < a.S; base += 32) {
        z = base + lane < a.S ? llb_span(a, base + lane) : LlbSpan{0, 0, 0};
        mine = llb_span_tiles(a, z, tile);
        p.total += __reduce_add_sync(0xffffffffu, mine);
    }
    p.blocks = min(grid, (p.total + least - 1) / least);
    p.t0 = p.t1 = 0;
    if (block >= p.blocks) return p;
    p.t0 = p.start(block);
    p.t1 = p.start(block + 1);
    int before = 0;
#pragma unroll 1
    for (int base = 0; base < a.S; base += 32) {
        if (a.S > 32) {
            z = base + lane < a.S ? llb_span(a, base + lane) : LlbSpan{0, 0, 0};
            mine = llb_span_tiles(a, z, tile);
        }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + sum > p.t0);
        if (past) {
            const int at = __ffs(past) - 1;
            p.job.s = base + at;
            p.job.begin = before + __shfl_sync(0xffffffffu, sum - mine, at);
            p.job.z.row = __shfl_sync(0xffffffffu, z.row, at);
            p.job.z.len = __shfl_sync(0xffffffffu, z.len, at);
            p.job.z.pos = __shfl_sync(0xffffffffu, z.pos, at);
            break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    p.job.first = 0;
#pragma unroll 1
    for (;;) {
        p.job.measure(a, tile);
        if (p.t0 < p.job.begin + (p.job.tiles + a.extra) * a.Hkv) break;
        p.job.begin += (p.job.tiles + a.extra) * a.Hkv;
        p.job.first += a.nodes;
    }
    p.job.kvh = (p.t0 - p.job.begin) / (p.job.tiles + a.extra);
    p.job.begin += p.job.kvh * (p.job.tiles + a.extra);
    return p;
}
// Where a job's partial result goes when the block [t0, t1) has not all of it: 0 or 1, or -1 when it has.
__device__ __forceinline__ int llb_part_of(const LlbPiece& p, const LlbJob& j) {
    if (j.begin < p.t0) return 0;
    return j.begin + j.tiles > p.t1 ? 1 : -1;
}

// What a key of a request received, onto what it had: nothing, if it is new.
__device__ __forceinline__ void llb_add_mass(const LlbSpanArgs& a, const LlbSpan& z, int s, int key, int kvh, float sum) {
    const int slot = key < z.pos + z.len ? llb_span_slot(a, s, key) : -1;
    if (slot < 0) return;
    const size_t at = (size_t)kvh * a.num_slots + slot;
    a.mass[at] = key < z.pos && a.mass_in ? a.mass_in[at] + sum : sum;
}

// (Minus infinity where everything that the row sees scores minus infinity: the weights are then 2^(-inf + inf), NaN, like the row's result.)
__device__ __forceinline__ float llb_lse(float m, float l) { return m + log2f(l); }
// What a row's sum of weights begins with, so that 1 / sum is what its weighted values are multiplied by: infinity, which the sum then
// stays, in a row that sees nothing (one of a tree's whose mask names none of the nodes, in a request that holds no keys) and gets zeros; 0 in
// all others, and where everything that such a row sees scores minus infinity 1 / 0 makes it NaN.
__device__ __forceinline__ float llb_first_sum(const LlbSpanArgs& a, const LlbSpan& z, int node) {
    if (!a.mask || z.pos > 0) return 0.0f;
    const unsigned long long* mask = a.mask + (size_t)(z.row + node) * a.words;
    int left = z.len;
#pragma unroll 1
    for (; left >= 64; left -= 64)
        if (*mask++) return 0.0f;
    return left > 0 && *mask << (64 - left) ? 0.0f : INFINITY;
}

// A job whose parts are to be joined, as the block that it begins in leaves it (parts 0: it has none).
struct LlbOpen {
    int parts, row, rows, kvh;      // blocks that have parts; first row of q, (row, head) pairs, kv head
};
__device__ __forceinline__ void llb_leave_open(const LlbSpanArgs& a, const LlbPiece& pc, const LlbJob& job, bool goes_on) {
    reinterpret_cast<int4*>(a.open)[blockIdx.x] = make_int4(goes_on ? pc.owner(job.begin + job.tiles - 1) - blockIdx.x + 1 : 0,
                                                            job.z.row + job.first, job.count(a) * a.group, job.kvh);
}

// Joins the parts of cut jobs and, for requests of one row (a.scores), adds up the weights that their keys received; `blocks` is the grid
// of the attention kernel, `tile` its keys a tile, `least` what it gave llb_piece.
int llb_span_join(const LlbSpanArgs& a, int dtype, int blocks, int tile, int least, cudaStream_t stream);

// ---- the weights that keys receive, of requests of several rows ------------------------------------------------------------------
// A job is a tile of keys of one request and kv head; the tiles of `nodes` rows that see any of them make the line that is cut among the
// blocks.  A job that a cut falls into leaves partial sums, which a second kernel adds up in the blocks' order.
struct LlbMassJob {
    LlbSpan z;
    int s, tile, kvh;
    int from, units, begin;     // first tile of rows that sees the keys, how many do, the job's place in the line
    __device__ __forceinline__ void measure(int keys, int nodes) {
        from = max(0, tile * keys - z.pos) / nodes;
        units = (z.len + nodes - 1) / nodes - from;
    }
    __device__ __forceinline__ int tiles(int keys) const { return z.len > 0 ? (z.pos + z.len + keys - 1) / keys : 0; }
    __device__ __forceinline__ void next(const LlbSpanArgs& a, int keys, int nodes) {
        begin += units;
        if (++kvh < a.Hkv) return;
        kvh = 0;
        ++tile;
#pragma unroll 1
        while (tile >= tiles(keys)) {
            z = llb_span(a, ++s);
            tile = 0;
        }
        measure(keys, nodes);
    }
};
struct LlbMassPiece {
    LlbPiece line;              // (its job is not used)
    LlbMassJob job;
};
__device__ __forceinline__ int llb_mass_units(const LlbSpanArgs& a, const LlbSpan& z, int keys, int nodes) {
    if (z.len == 0) return 0;
    const int rows = (z.len + nodes - 1) / nodes, whole = z.pos / keys + 1, tiles = (z.pos + z.len + keys - 1) / keys;
    int n = whole * rows;          // (whole <= tiles: the first row sees key pos)
#pragma unroll 1
    for (int i = whole; i < tiles; ++i) n += rows - (i * keys - z.pos) / nodes;
    return n * a.Hkv;
}
__device__ __forceinline__ LlbMassPiece llb_mass_piece(const LlbSpanArgs& a, int keys, int nodes, int block, int grid, int lane) {
    LlbMassPiece m;
    LlbPiece& p = m.line;
    int mine = 0;
    p.total = 0;
#pragma unroll 1
    for (int base = 0; base < a.S; base += 32) {
        mine = base + lane < a.S ? llb_mass_units(a, llb_span(a, base + lane), keys, nodes) : 0;
        p.total += __reduce_add_sync(0xffffffffu, mine);
    }
    p.blocks = min(grid, (p.total + 1) / 2);
    p.t0 = p.t1 = 0;
    if (block >= p.blocks) return m;
    p.t0 = p.start(block);
    p.t1 = p.start(block + 1);
    int before = 0;
#pragma unroll 1
    for (int base = 0; base < a.S; base += 32) {
        if (a.S > 32) mine = base + lane < a.S ? llb_mass_units(a, llb_span(a, base + lane), keys, nodes) : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + sum > p.t0);
        if (past) {
            const int at = __ffs(past) - 1;
            m.job.s = base + at;
            m.job.begin = before + __shfl_sync(0xffffffffu, sum - mine, at);
            break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    m.job.z = llb_span(a, m.job.s);
    m.job.tile = 0;
#pragma unroll 1
    for (;;) {
        m.job.measure(keys, nodes);
        if (p.t0 < m.job.begin + m.job.units * a.Hkv) break;
        m.job.begin += m.job.units * a.Hkv;
        ++m.job.tile;
    }
    m.job.kvh = (p.t0 - m.job.begin) / m.job.units;
    m.job.begin += m.job.kvh * m.job.units;
    return m;
}
// What the block that a job begins in leaves of it: how many blocks have parts (0: it has no such job), request, tile and kv head.
__device__ __forceinline__ void llb_leave_open_mass(const LlbSpanArgs& a, const LlbPiece& line, const LlbMassJob& job, bool goes_on) {
    reinterpret_cast<int4*>(a.open)[blockIdx.x] =
        goes_on ? make_int4(line.owner(job.begin + job.units - 1) - blockIdx.x + 1, job.s, job.tile, job.kvh) : make_int4(0, 0, 0, 0);
}

// The tensor-core kernels (span_attention_tcgen05.cu): whether they take a call, how many rows of a request fill 128 pairs, the attention
// (a.nodes twice that many, a.rows 2 x 128), and the weights of keys (part: 2 * blocks * 128 floats).
bool llb_span_tc_takes(const LlbSpanArgs& a, const void* q, const void* k, const void* v, const void* out);
int llb_span_tc_pairs(int group);
int llb_span_attention_tc(const LlbSpanArgs& a, const void* q, const void* k, const void* v, int blocks, int* error_flag, cudaStream_t stream);
int llb_span_mass_tc(const LlbSpanArgs& a, const void* q, const void* k, float* part, int blocks, int* error_flag, cudaStream_t stream);
