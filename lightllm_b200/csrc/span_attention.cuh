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
// A job that a cut falls into leaves partial results (O, m, l); the block that leaves the last of them joins all, in the order of the
// blocks, so the result does not depend on which block that is.  Everything is worked out on the device: a captured graph serves
// other lengths.
#pragma once
#include "common.cuh"

constexpr int LLB_SPAN_BLOCKS = 512;          // blocks of a kernel at most

struct LlbSpanArgs {
    const int* span_row;             // [S]
    const int* span_len;
    const int* span_pos;
    const int* table;                // [S, max_pages]
    int S, T, max_pages, page_size, max_len, num_slots;
    int Hq, Hkv, hd, group;
    const unsigned long long* mask;  // tree: [T, words]; null: causal
    int words;
    float scale_log2e;               // scores are kept in base-2 units
    void* out;                       // [T, Hq, hd]
    float* lse;                      // [T, Hq] or null: log2 of the sum of 2^score; +infinity in a row that sees nothing
    float* scores;                   // [score_tiles, group, keys a tile] or null: the scores of requests of one row, tile by tile of the line
    int score_tiles;
    const float* mass_in;            // [Hkv, num_slots] or null: zeros
    float* mass;                     // [Hkv, num_slots] or null: what joins a job of a request of one row adds up its scores' weights
    float* part_o;                   // [2 * blocks, rows, hd]: what a block has of a job that began before it (0) and goes on after it (1)
    float* part_ml;                  // [2 * blocks, rows, 2]
    unsigned* arrived;               // [blocks] how many of a job's parts there are, by the block that it begins in; zero before and after
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
    const int page = a.table[(size_t)s * a.max_pages + key / a.page_size];
    const long long slot = (long long)page * a.page_size + key % a.page_size;
    return page >= 0 && slot < a.num_slots ? (int)slot : -1;
}

// A job and its tiles' place in the line of all tiles.
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
        begin += tiles;
        if (++kvh < a.Hkv) return;
        kvh = 0;
        first += a.nodes;
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
};
__device__ __forceinline__ int llb_span_tiles(const LlbSpanArgs& a, const LlbSpan& z, int tile) {
    int n = 0;
    if (z.len > 0 && a.mask) n = (z.len + a.nodes - 1) / a.nodes * ((z.pos + z.len + tile - 1) / tile);
    else
        for (int c = 0; c < z.len; c += a.nodes) n += (llb_span_keys(a, z, c + a.nodes) + tile - 1) / tile;
    return n * a.Hkv;
}
// By one whole warp; every lane gets the answer.  A block has `least` tiles or more where there are enough.
__device__ __forceinline__ LlbPiece llb_piece(const LlbSpanArgs& a, int tile, int block, int grid, int least, int lane) {
    LlbPiece p;
    LlbSpan z = {0, 0, 0};
    int mine = 0;
    p.total = 0;
    for (int base = 0; base < a.S; base += 32) {
        z = base + lane < a.S ? llb_span(a, base + lane) : LlbSpan{0, 0, 0};
        mine = llb_span_tiles(a, z, tile);
        p.total += __reduce_add_sync(0xffffffffu, mine);
    }
    p.blocks = min(grid, (p.total + least - 1) / least);
    p.t0 = p.t1 = 0;
    if (block >= p.blocks) return p;
    p.t0 = (int)((long long)p.total * block / p.blocks);
    p.t1 = (int)((long long)p.total * (block + 1) / p.blocks);
    int before = 0;
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
    for (;;) {
        p.job.measure(a, tile);
        if (p.t0 < p.job.begin + p.job.tiles * a.Hkv) break;
        p.job.begin += p.job.tiles * a.Hkv;
        p.job.first += a.nodes;
    }
    p.job.kvh = (p.t0 - p.job.begin) / p.job.tiles;
    p.job.begin += p.job.kvh * p.job.tiles;
    return p;
}
// Which block has tile t of the line.
__device__ __forceinline__ int llb_piece_owner(const LlbPiece& p, int t) {
    return (int)(((long long)(t + 1) * p.blocks + p.total - 1) / p.total) - 1;
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

__device__ __forceinline__ float llb_lse(float m, float l) { return l == 0.0f ? INFINITY : m + log2f(l); }
// What a row's sum of weighted values is multiplied by: 0 in a row that sees nothing; where everything that it sees scores minus infinity
// it is 1 / 0, and the row is NaN.
__device__ __forceinline__ float llb_inverse(float m, float l, int pos) { return l > 0.0f || m != -INFINITY || pos > 0 ? 1.0f / l : 0.0f; }

// Joins rows of a job from its parts, PB parts of RU rows at a time so that 16 loads of 16 bytes are on their way a thread (what bounds
// a joining block is the latency of the second-level cache).  TPR threads have a row, four dimensions each (and the next 4 * TPR).
// Rows base .. base + rows - 1 of the job; w_s: the parts' factors for them [parts, rows], 2^(m - M) / L.
template <typename T, int TPR, int PB, int RU>
__device__ __forceinline__ void llb_join_rows(const LlbSpanArgs& a, const LlbJob& job, int from, int parts, int base, int rows, const float* w_s, int tid) {
    constexpr int RPP = 256 / TPR;
    const int hd = a.hd, pieces = (hd + 3) / 4;
    const size_t next = (size_t)2 * a.rows * hd;                                     // from a part to the next
    const float* first = a.part_o + (size_t)(from * 2) * a.rows * hd;                // (part 0 is the second one of its block)
    for (int piece = tid % TPR; piece < pieces; piece += TPR) {
        const int d = piece * 4;
        const bool whole = hd % 4 == 0;
        for (int r0 = tid / TPR; r0 < rows; r0 += RPP * RU) {
            float4 x[RU];
#pragma unroll
            for (int u = 0; u < RU; ++u) x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int b0 = 0; b0 < parts; b0 += PB) {
                float4 v[RU][PB];
#pragma unroll
                for (int u = 0; u < RU; ++u)
#pragma unroll
                    for (int e = 0; e < PB; ++e) {
                        const int r = r0 + u * RPP, b = b0 + e;
                        v[u][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (r >= rows || b >= parts) continue;
                        const float* o = first + (b == 0 ? (size_t)a.rows * hd : b * next) + (size_t)(base + r) * hd + d;
                        if (whole) v[u][e] = __ldcg(reinterpret_cast<const float4*>(o));
                        else {
                            v[u][e].x = __ldcg(o);
                            if (d + 1 < hd) v[u][e].y = __ldcg(o + 1);
                            if (d + 2 < hd) v[u][e].z = __ldcg(o + 2);
                            if (d + 3 < hd) v[u][e].w = __ldcg(o + 3);
                        }
                    }
#pragma unroll
                for (int u = 0; u < RU; ++u)
#pragma unroll
                    for (int e = 0; e < PB; ++e) {
                        const int r = r0 + u * RPP, b = b0 + e;
                        if (r >= rows || b >= parts) continue;
                        const float w = w_s[b * rows + r];
                        x[u].x = fmaf(w, v[u][e].x, x[u].x);
                        x[u].y = fmaf(w, v[u][e].y, x[u].y);
                        x[u].z = fmaf(w, v[u][e].z, x[u].z);
                        x[u].w = fmaf(w, v[u][e].w, x[u].w);
                    }
            }
#pragma unroll
            for (int u = 0; u < RU; ++u) {
                const int r = r0 + u * RPP;
                if (r >= rows) continue;
                const int node = (base + r) / a.group;
                T* dst = (T*)a.out + ((size_t)(job.z.row + job.first + node) * a.Hq + job.kvh * a.group + base + r - node * a.group) * hd + d;
                if (whole && sizeof(T) == 2 && ((uintptr_t)dst & 7) == 0) {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[u].x, x[u].y), hi = __floats2bfloat162_rn(x[u].z, x[u].w);
                    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
                    continue;
                }
                dst[0] = llb_from_float<T>(x[u].x);
                if (d + 1 < hd) dst[1] = llb_from_float<T>(x[u].y);
                if (d + 2 < hd) dst[2] = llb_from_float<T>(x[u].z);
                if (d + 3 < hd) dst[3] = llb_from_float<T>(x[u].w);
            }
        }
    }
}

// The end of a job, by the 256 threads that have its rows (tid 0 .. 255; `barrier` is one of theirs alone; `room` is `floats` of shared
// memory, at least 2 a row of the job and one a row for each of four parts).  `part` says what this block has: a part, which is in part_o
// and part_ml already, or (-1) the whole job, whose rows are written and whose m and l are in room.  The last part's block joins the rows:
//     out = sum_b 2^(m_b - M) O_b / sum_b 2^(m_b - M) l_b
// and whoever has a request's only row then adds up the weights of its keys, if a.mass asks for them.
template <typename T, int TILE, int TPR, typename Barrier>
__device__ __forceinline__ void llb_finish_job(const LlbSpanArgs& a, const LlbPiece& pc, const LlbJob& job, int part, float* room, int floats,
                                               int* flag, int tid, const Barrier& barrier) {
    const bool adds = a.mass && a.scores && job.z.len == 1;
    if (part < 0 && !adds) return;
    const int rows = job.count(a) * a.group;
    barrier();
    if (part >= 0) {
        const int from = llb_piece_owner(pc, job.begin), parts = llb_piece_owner(pc, job.begin + job.tiles - 1) - from + 1;
        if (tid == 0) {
            __threadfence();             // all threads' parts (and scores), which the barrier has put before this, come before the arrival
            *flag = atomicInc(a.arrived + from, parts - 1) == (unsigned)parts - 1;          // (back to zero at the last)
            __threadfence();
        }
        barrier();
        if (!*flag) return;
        // the factors of all parts of all rows, so many rows at a time as there is room for (all of them but for very long lines of parts)
        float* ml_s = room;              // [rows] m and l
        float* w_s = room + 2 * rows;
        const int at_once = max(1, min(rows, (floats - 2 * rows) / parts));
        const float2* first = reinterpret_cast<const float2*>(a.part_ml) + (size_t)(from * 2) * a.rows;
        for (int base = 0; base < rows; base += at_once) {
            const int count = min(at_once, rows - base);
            if (base > 0) barrier();
            for (int r = tid; r < count; r += 256) {
                const float2* ml = first + base + r;
                float M = -INFINITY, L = 0.0f;
#pragma unroll 8
                for (int b = 0; b < parts; ++b) M = fmaxf(M, __ldcg(ml + (b == 0 ? 1 : 2 * b) * (size_t)a.rows).x);
#pragma unroll 8
                for (int b = 0; b < parts; ++b) {
                    const float2 x = __ldcg(ml + (b == 0 ? 1 : 2 * b) * (size_t)a.rows);
                    // (a part without visible keys has m = -infinity, l = 0 and O = 0; a NaN of another one stays)
                    const float w = x.x == -INFINITY ? 1.0f : exp2f(x.x - M);
                    w_s[b * count + r] = w;
                    L = fmaf(w, x.y, L);
                }
                const float inv = llb_inverse(M, L, job.z.pos);
                for (int b = 0; b < parts; ++b) w_s[b * count + r] *= inv;
                ml_s[2 * (base + r)] = M;
                ml_s[2 * (base + r) + 1] = L;
                const int node = (base + r) / a.group;
                if (a.lse)
                    a.lse[(size_t)(job.z.row + job.first + node) * a.Hq + job.kvh * a.group + base + r - node * a.group] = llb_lse(M, L);
            }
            barrier();
            if (parts <= 2) llb_join_rows<T, TPR, 2, 8>(a, job, from, parts, base, count, w_s, tid);
            else if (parts <= 4) llb_join_rows<T, TPR, 4, 4>(a, job, from, parts, base, count, w_s, tid);
            else llb_join_rows<T, TPR, 8, 2>(a, job, from, parts, base, count, w_s, tid);
        }
    }
    if (!adds) return;
    for (int key = tid; key <= job.z.pos; key += 256) {
        const int tile = job.begin + key / TILE;
        float sum = 0.0f;
        if (tile < a.score_tiles)
            for (int g = 0; g < a.group; ++g)
                sum += exp2f(__ldcg(a.scores + ((size_t)tile * a.group + g) * TILE + key % TILE) - room[2 * g]) / room[2 * g + 1];
        llb_add_mass(a, job.z, job.s, key, job.kvh, sum);
    }
}

// The tensor-core kernels (span_attention_tcgen05.cu): whether they take a call, how many rows of a request fill 128 pairs, the attention
// (a.nodes twice that many, a.rows 2 x 128), and the weights of keys (part: 2 * blocks * 128 floats).
bool llb_span_tc_takes(const LlbSpanArgs& a, const void* q, const void* k, const void* v, const void* out);
int llb_span_tc_pairs(int group);
int llb_span_attention_tc(const LlbSpanArgs& a, const void* q, const void* k, const void* v, int blocks, int* error_flag, cudaStream_t stream);
int llb_span_mass_tc(const LlbSpanArgs& a, const void* q, const void* k, float* part, int blocks, int* error_flag, cudaStream_t stream);
