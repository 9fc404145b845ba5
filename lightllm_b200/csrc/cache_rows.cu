// Kernels that move rows of the paged cache: the commit of confirmed drafted tokens, and eviction by accumulated attention weight.
// Both work on all layers of a group of planes at once: keys and values [layers, slots, kv heads, head size].
#include "cache_calls.h"
#include "common.cuh"
#include "memory_ranges.h"
#include "shared_memory.h"
#include "tcgen05_common.cuh"

namespace {

// The kernel before has completed.  The next one is not let in early, as other kernels of the library do: these move keys that are not new,
// and decode attention reads such keys before it waits.  It may be the next one and begin as soon as the last block here has ended, when only
// its own wait would promise it what was written: so a thread that has moved rows ends with before_next().
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// What this thread has written is in the memory that all multiprocessors read.
__device__ __forceinline__ void before_next() { __threadfence(); }

// The cache row of a place of a request, or -1 for a page that is none of the cache's: such a place is neither read nor written.
__device__ __forceinline__ int slot_of(const int* table, int page_size, int num_slots, int place) {
    const int page = table[place / page_size];
    const long long slot = (long long)page * page_size + place % page_size;
    return page >= 0 && slot < num_slots ? (int)slot : -1;
}

// ---- the confirmed drafted tokens --------------------------------------------------------------------------------------------
// A request's nodes are its rows: node 0 is the newest confirmed token, every other node continues its parent (of a lower number)
// with a drafted token.  What the model chooses behind a node confirms the first of the node's children with that token:
//     path[0] = 0,   path[d + 1] = the lowest c with parents[c] = path[d] and tokens[c] = targets[path[d]]
// The keys and values of node path[d] lie at place pos + path[d] and belong to pos + d.  path rises strictly, so path[d] >= d: a row
// never moves onto one that is still to be read when the rows move in the path's order, and a thread that moves the same 16 bytes of
// every row needs no meeting with others; it reads eight rows ahead.
// Every block works out the path for itself (a warp looks at 32 nodes at a time), which is less than a second launch would take.
constexpr int COMMIT_THREADS = 128;
constexpr int COMMIT_MAX_PATH = 1024;
constexpr int COMMIT_AHEAD = 8;
struct CommitParams {
    const int* tokens;
    const int* parents;
    const int* targets;
    const int* span_row;
    const int* span_len;
    const int* span_pos;
    const int* table;
    char* k;
    char* v;
    int* path;
    int* count;
    int* next;
    int S, T, L, max_pages, page_size, num_slots, width;
    int row_units;               // of one slot's row of K (or V), in units of the copies
    int layers_a_block;
};

template <typename U>
__global__ void __launch_bounds__(COMMIT_THREADS) tree_commit_kernel(const CommitParams p) {
    __shared__ int path_s[COMMIT_MAX_PATH];
    __shared__ int slot_s[2][COMMIT_MAX_PATH];
    __shared__ int count_s;
    after_previous();
    const int s = blockIdx.x, lane = threadIdx.x & 31;
    const int row = p.span_row[s], pos = max(p.span_pos[s], 0);
    int n = min(min(p.span_len[s], p.T - row), p.max_pages * p.page_size - pos);
    if (row < 0 || n < 0) n = 0;
    if (threadIdx.x < 32) {
        int count = 0, cur = 0;
        if (n > 0) {
            if (lane == 0) path_s[0] = 0;
            count = 1;
            while (count < p.width) {
                const int want = p.targets[row + cur];
                int child = -1;
                for (int c0 = cur + 1; c0 < n; c0 += 32) {
                    const int c = c0 + lane;
                    const unsigned fits = __ballot_sync(0xffffffffu, c < n && p.parents[row + c] == cur && p.tokens[row + c] == want);
                    if (fits) {
                        child = c0 + __ffs(fits) - 1;
                        break;
                    }
                }
                if (child < 0) break;
                cur = child;
                if (lane == 0) path_s[count] = cur;
                ++count;
            }
        }
        if (lane == 0) count_s = count;
        if (blockIdx.y == 0) {
            __syncwarp();
            for (int d = lane; d < p.width; d += 32) p.path[(size_t)s * p.width + d] = d < count ? path_s[d] : -1;
            if (lane == 0) {
                p.count[s] = count;
                p.next[s] = count > 0 ? p.targets[row + cur] : -1;
            }
        }
    }
    __syncthreads();
    const int count = count_s;
    const int* table = p.table + (size_t)s * p.max_pages;
    for (int d = threadIdx.x; d < count; d += COMMIT_THREADS) {
        slot_s[0][d] = path_s[d] == d ? -1 : slot_of(table, p.page_size, p.num_slots, pos + path_s[d]);
        slot_s[1][d] = path_s[d] == d ? -1 : slot_of(table, p.page_size, p.num_slots, pos + d);
    }
    __syncthreads();
    const int units = 2 * p.row_units;
    for (int i = threadIdx.x; i < p.layers_a_block * units; i += COMMIT_THREADS) {
        const int layer = blockIdx.y * p.layers_a_block + i / units;
        if (layer >= p.L) break;
        const int u = i % units;
        U* base = (U*)(u < p.row_units ? p.k : p.v) + (size_t)layer * p.num_slots * p.row_units + (u < p.row_units ? u : u - p.row_units);
        for (int d0 = 1; d0 < count; d0 += COMMIT_AHEAD) {
            U x[COMMIT_AHEAD];
#pragma unroll
            for (int e = 0; e < COMMIT_AHEAD; ++e)
                if (d0 + e < count && slot_s[0][d0 + e] >= 0) x[e] = base[(size_t)slot_s[0][d0 + e] * p.row_units];
#pragma unroll
            for (int e = 0; e < COMMIT_AHEAD; ++e)
                if (d0 + e < count && slot_s[0][d0 + e] >= 0 && slot_s[1][d0 + e] >= 0) base[(size_t)slot_s[1][d0 + e] * p.row_units] = x[e];
        }
    }
    before_next();
}

// ---- eviction ------------------------------------------------------------------------------------------------------------------
// For every layer, request and kv head: of the n places that are held the `budget` that are worth most stay, a place's worth being
// the weight that its key has received, above everything else the places of the first and of the latest positions, and of equal
// ones the lowest place.  What stays lies in the places below the budget afterwards: the dropped ones among them (holes, in rising
// order) take the keys, values, weights and positions of those that stay beyond it (in rising order).  Attention does not ask for
// the order of its keys (they carry their rotation), so nothing else moves: as many rows as there are holes instead of nearly all.
//
// A block takes one (layer, request, kv head), or as many as fill the device share its moves.  A thread has up to 8 or 32 places, all asked for at once (what a block's time is made of is
// trips to memory, 0.6 us each): their cache rows and their worth as whole numbers in the floats' order stay in registers.  The
// budget's threshold is found digit by digit from the top, 11, 11 and 10 bits, by counting, the dropping of a single place by one search for
// the least.  The places that stay become a bit each, which gives holes and fillers their numbers by counting bits; the moves
// are then dealt evenly to all threads, 16 bytes at a time.  Tables of more places go through a kernel that keeps the worths that fit in
// shared memory and reads the rest again.
constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_LIST = 2048;             // moves that are listed at a time
constexpr int EV_MAX_PLACES = 1 << 20;
struct EvictParams {
    char* k;
    char* v;
    const float* mass;                    // [L, Hkv, num_slots]
    const int* positions;
    float* mass_out;
    int* positions_out;
    const int* lengths;                   // [S] places that are held
    const int* ends;                      // [S] position of the request's next token
    const int* table;
    int S, max_pages, page_size, num_slots, Hkv, budget, first, latest;
    int head_units;                       // of one head's row of K (or V), in units of the copies
    int cache_places;                     // as many worths as shared memory holds
    int parts;                            // blocks that share the moves of one (layer, request, kv head), a power of two
};

__device__ __forceinline__ unsigned order_of(float f) {
    if (f != f) return 0xfffffffeu;                      // NaN: above infinity
    const unsigned u = __float_as_uint(f + 0.0f);        // (-0 becomes +0)
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The listed moves begin .. end - 1 of one (layer, kv head): rows of K and V, 16 bytes a thread and AHEAD of them on their way, then weights and positions.
template <typename U>
__device__ __forceinline__ void move_rows(const EvictParams& p, size_t plane, int layer, int h, const unsigned (&list)[2][EV_LIST], unsigned begin, unsigned end) {
    constexpr int AHEAD = 4;
    const unsigned units = 2 * p.head_units, total = end * units;
    const size_t stride = (size_t)p.Hkv * p.head_units, base = (size_t)layer * p.num_slots * stride + (size_t)h * p.head_units;
    const int shift = (units & (units - 1)) == 0 ? 31 - __clz(units) : -1;          // (heads of 64 and 128: no division)
    for (unsigned i0 = begin * units + threadIdx.x; i0 < total; i0 += EV_THREADS * AHEAD) {
        U x[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const unsigned i = i0 + e * EV_THREADS;
            if (i >= total) continue;
            const unsigned m = shift >= 0 ? i >> shift : i / units, u = i - m * units;
            const int src = (int)list[1][m];
            const U* from = (const U*)(u < (unsigned)p.head_units ? p.k : p.v) + base + (u < (unsigned)p.head_units ? u : u - p.head_units);
            if (src >= 0) x[e] = from[(size_t)src * stride];
        }
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const unsigned i = i0 + e * EV_THREADS;
            if (i >= total) continue;
            const unsigned m = shift >= 0 ? i >> shift : i / units, u = i - m * units;
            const int src = (int)list[1][m], dst = (int)list[0][m];
            U* to = (U*)(u < (unsigned)p.head_units ? p.k : p.v) + base + (u < (unsigned)p.head_units ? u : u - p.head_units);
            if (src >= 0 && dst >= 0) to[(size_t)dst * stride] = x[e];
        }
    }
    for (unsigned m = begin + threadIdx.x; m < end; m += EV_THREADS) {
        const int src = (int)list[1][m], dst = (int)list[0][m];
        if (src < 0 || dst < 0) continue;
        p.mass_out[plane + dst] = p.mass[plane + src];
        p.positions_out[plane + dst] = p.positions[plane + src];
    }
}

// Where `wanted` of those whose digits above this one are `prefix` end, counted from the top: hist holds how many have each value of
// the digit.  found: the prefix with this digit, how many of its bearers are wanted, how many there are.
__device__ __forceinline__ void find_digit(const unsigned (&hist)[EV_BINS], unsigned prefix, unsigned wanted, int shift, unsigned (&warp_s)[EV_WARPS][2],
                                           unsigned (&found)[3]) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int PER = EV_BINS / EV_THREADS;
    const int top = EV_BINS - 1 - tid * PER;
    unsigned mine = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) mine += hist[top - b];
    unsigned sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
    }
    if (lane == 31) warp_s[warp][0] = sum;
    __syncthreads();
    unsigned above = sum - mine;
    for (int w = 0; w < warp; ++w) above += warp_s[w][0];
    if (above < wanted && above + mine >= wanted) {
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            const unsigned c = hist[top - b];
            if (above < wanted && above + c >= wanted) {
                found[0] = prefix | ((unsigned)(top - b) << shift);
                found[1] = wanted - above;
                found[2] = c;
            }
            above += c;
        }
    }
    __syncthreads();
}

// Exclusive sums of `words` counts (two to a word: low and high half) by the first warp; everyone has them and the totals afterwards.
template <int WORDS> __device__ __forceinline__ void scan_words(unsigned (&count)[WORDS], unsigned& total_s, int words) {
    __syncthreads();
    if (threadIdx.x < 32) {
        unsigned before = 0;
        for (int w0 = 0; w0 < words; w0 += 32) {
            const int w = w0 + threadIdx.x;
            const unsigned mine = w < words ? count[w] : 0u;
            unsigned sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffffu, sum, o);
                if ((int)threadIdx.x >= o) sum += x;
            }
            if (w < words) count[w] = before + sum - mine;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (threadIdx.x == 0) total_s = before;
    }
    __syncthreads();
}

// SHARED: the p.parts blocks of a cluster take one (layer, request, kv head).
template <typename U, int PER, bool SHARED>
__global__ void __launch_bounds__(EV_THREADS, PER <= 8 ? 3 : 1) cache_evict_kernel(const EvictParams p) {
    constexpr int WORDS = PER * EV_WARPS;
    __shared__ unsigned hist[EV_BINS];
    __shared__ unsigned list_s[2][EV_LIST];
    __shared__ unsigned warp_s[EV_WARPS][2], word_s[WORDS];
    __shared__ unsigned long long least_s[EV_WARPS];
    __shared__ unsigned found_s[3], total_s;
    after_previous();
    const int parts = SHARED ? p.parts : 1, part = blockIdx.x & (parts - 1), both = blockIdx.x / parts;
    const int s = both / p.Hkv, h = both - s * p.Hkv, layer = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = max(0, min(p.lengths[s], p.max_pages * p.page_size)), budget = p.budget;
    const int from = p.ends[s] - p.latest;
    const int* table = p.table + (size_t)s * p.max_pages;
    const size_t plane = ((size_t)layer * p.Hkv + h) * p.num_slots;
    const bool apart = p.mass_out != p.mass;
    const int page_shift = (p.page_size & (p.page_size - 1)) == 0 ? 31 - __clz(p.page_size) : -1;
    if (n <= budget && !apart) return;
    // place k * EV_THREADS + tid: word k * EV_WARPS + warp of the bits, bit `lane`
    int slot[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * EV_THREADS + tid;
        slot[k] = -1;
        if (i < n) {
            const int page_of = page_shift >= 0 ? i >> page_shift : i / p.page_size;
            const int page = table[page_of];
            const long long at = (long long)page * p.page_size + (i - page_of * p.page_size);
            if (page >= 0 && at < p.num_slots) slot[k] = (int)at;
        }
    }
    // the weights and positions of the places that stay where they are
    auto copy = [&](auto stays) {
        if (!apart) return;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            if (k * EV_THREADS >= min(n, budget) || (k & (parts - 1)) != part || slot[k] < 0 || !stays(k)) continue;
            p.mass_out[plane + slot[k]] = p.mass[plane + slot[k]];
            p.positions_out[plane + slot[k]] = p.positions[plane + slot[k]];
        }
    };
    if (n <= budget) {
        copy([&](int) { return true; });
        return;
    }
    unsigned worth[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        worth[k] = 0u;
        if (slot[k] < 0) continue;
        const int pos = p.positions[plane + slot[k]];
        worth[k] = pos < p.first || pos >= from ? 0xffffffffu : order_of(p.mass[plane + slot[k]]);
    }

    if (n == budget + 1) {
        // one place goes: the least worth, of equal ones the highest place
        if (part > 0 && !apart) return;          // (a single move, and it may write what this block reads)
        unsigned long long least = ~0ull;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = k * EV_THREADS + tid;
            const unsigned long long x = ((unsigned long long)worth[k] << 32) | (unsigned)(n - 1 - i);
            if (i < n && x < least) least = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long x = __shfl_xor_sync(0xffffffffu, least, o);
            least = x < least ? x : least;
        }
        if (lane == 0) least_s[warp] = least;
        __syncthreads();
        least = least_s[0];
#pragma unroll
        for (int w = 1; w < EV_WARPS; ++w) least = least_s[w] < least ? least_s[w] : least;
        const int hole = n - 1 - (int)(unsigned)least;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = k * EV_THREADS + tid;
            if (i == hole) list_s[0][0] = slot[k];
            if (i == n - 1) list_s[1][0] = slot[k];
        }
        __syncthreads();
        if (hole != n - 1 && part == 0) move_rows<U>(p, plane, layer, h, list_s, 0, 1);
        copy([&](int k) { return k * EV_THREADS + tid < budget && k * EV_THREADS + tid != hole; });
        before_next();
        return;
    }

    // the blocks of a cluster write, in place, what the others have read
    if (SHARED && !apart) t5::cluster_sync_all();

    // the threshold: the budget-th largest worth, and how many of its equals stay
    unsigned prefix = 0, wanted = budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
        for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k)
            // (64 bits: a shift by 32 would be none)
            if (k * EV_THREADS + tid < n && ((unsigned long long)(worth[k] ^ prefix) >> (shift + width)) == 0)
                atomicAdd(&hist[(worth[k] >> shift) & ((1u << width) - 1u)], 1u);
        __syncthreads();
        find_digit(hist, prefix, wanted, shift, warp_s, found_s);
        prefix = found_s[0];
        wanted = found_s[1];
    }
    const int words = (n + 31) / 32;
    unsigned stays = 0;          // a bit for each of the thread's places
    if (found_s[2] == wanted) {
#pragma unroll
        for (int k = 0; k < PER; ++k) stays |= (unsigned)(k * EV_THREADS + tid < n && worth[k] >= prefix) << k;
    } else {
        // of equals the lowest places stay: they are numbered
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const unsigned same = __ballot_sync(0xffffffffu, k * EV_THREADS + tid < n && worth[k] == prefix);
            if (lane == 0) word_s[k * EV_WARPS + warp] = __popc(same);
        }
        scan_words(word_s, total_s, words);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const bool held = k * EV_THREADS + tid < n;
            const unsigned same = __ballot_sync(0xffffffffu, held && worth[k] == prefix);
            const bool on = held && (worth[k] > prefix ||
                                     (worth[k] == prefix && word_s[k * EV_WARPS + warp] + __popc(same & ((1u << lane) - 1u)) < wanted));
            stays |= (unsigned)on << k;
        }
        __syncthreads();
    }
    // numbers of the holes (low half of a count) and of those that fill them (high half)
    auto is_hole = [&](int k) { return k * EV_THREADS + tid < budget && !((stays >> k) & 1u); };
    auto fills = [&](int k) { return k * EV_THREADS + tid >= budget && ((stays >> k) & 1u); };
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const unsigned a = __ballot_sync(0xffffffffu, is_hole(k)), b = __ballot_sync(0xffffffffu, fills(k));
        if (lane == 0) word_s[k * EV_WARPS + warp] = __popc(a) | (__popc(b) << 16);
    }
    scan_words(word_s, total_s, words);
    const unsigned moves = total_s & 0xffffu;
    for (unsigned m0 = 0; m0 < moves; m0 += EV_LIST) {
        const unsigned count = min((unsigned)EV_LIST, moves - m0);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const unsigned a = __ballot_sync(0xffffffffu, is_hole(k)), b = __ballot_sync(0xffffffffu, fills(k));
            const unsigned under = (1u << lane) - 1u, before = word_s[k * EV_WARPS + warp];
            const unsigned hr = (before & 0xffffu) + __popc(a & under) - m0, fr = (before >> 16) + __popc(b & under) - m0;
            if (is_hole(k) && hr < count) list_s[0][hr] = slot[k];
            if (fills(k) && fr < count) list_s[1][fr] = slot[k];
        }
        __syncthreads();
        move_rows<U>(p, plane, layer, h, list_s, count * part / parts, count * (part + 1) / parts);
        __syncthreads();
    }
    copy([&](int k) { return k * EV_THREADS + tid < budget && ((stays >> k) & 1u); });
    before_next();
}

template <typename U>
__global__ void __launch_bounds__(EV_THREADS) cache_evict_any_kernel(const EvictParams p) {
    extern __shared__ unsigned ev_sm[];
    __shared__ unsigned hist[EV_BINS];
    __shared__ unsigned list_s[2][EV_LIST];
    __shared__ unsigned warp_s[EV_WARPS][2];
    __shared__ unsigned found_s[3];
    after_previous();
    const int s = blockIdx.x / p.Hkv, h = blockIdx.x - s * p.Hkv, layer = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = max(0, min(p.lengths[s], p.max_pages * p.page_size)), budget = p.budget;
    const int* table = p.table + (size_t)s * p.max_pages;
    const size_t plane = ((size_t)layer * p.Hkv + h) * p.num_slots;
    const bool apart = p.mass_out != p.mass;
    unsigned* bits = ev_sm;                              // [words] places that stay
    const int words = (n + 31) / 32;
    unsigned* worth_s = ev_sm + (p.max_pages * p.page_size + 31) / 32;
    if (n <= budget) {
        if (apart)
            for (int i = tid; i < n; i += EV_THREADS) {
                const int slot = slot_of(table, p.page_size, p.num_slots, i);
                if (slot < 0) continue;
                p.mass_out[plane + slot] = p.mass[plane + slot];
                p.positions_out[plane + slot] = p.positions[plane + slot];
            }
        return;
    }
    const int from = p.ends[s] - p.latest;
    auto compute = [&](int i) -> unsigned {
        const int slot = slot_of(table, p.page_size, p.num_slots, i);
        if (slot < 0) return 0u;
        const int pos = p.positions[plane + slot];
        if (pos < p.first || pos >= from) return 0xffffffffu;
        return order_of(p.mass[plane + slot]);
    };
    const bool cached = n <= p.cache_places;
    auto worth = [&](int i) -> unsigned { return cached ? worth_s[i] : compute(i); };

    // the threshold: the budget-th largest worth, and how many of its equals stay
    unsigned prefix = 0, wanted = budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
        for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += EV_THREADS) {
            const unsigned x = pass == 0 ? compute(i) : worth(i);
            if (pass == 0 && cached) worth_s[i] = x;
            // (64 bits: a shift by 32 would be none)
            if (((unsigned long long)(x ^ prefix) >> (shift + width)) == 0) atomicAdd(&hist[(x >> shift) & ((1u << width) - 1u)], 1u);
        }
        __syncthreads();
        find_digit(hist, prefix, wanted, shift, warp_s, found_s);
        prefix = found_s[0];
        wanted = found_s[1];
    }
    // a bit for every place that stays: a warp takes words in a row, so that equals are counted in the places' order
    const int per_warp = (words + EV_WARPS - 1) / EV_WARPS;
    const int w0 = min(words, warp * per_warp), w1 = min(words, w0 + per_warp);
    unsigned equals = 0;
    for (int w = w0; w < w1; ++w) {
        const int i = w * 32 + lane;
        equals += __popc(__ballot_sync(0xffffffffu, i < n && worth(i) == prefix));
    }
    if (lane == 0) warp_s[warp][1] = equals;
    __syncthreads();
    unsigned before = 0;
    for (int w = 0; w < warp; ++w) before += warp_s[w][1];
    for (int w = w0; w < w1; ++w) {
        const int i = w * 32 + lane;
        const unsigned x = i < n ? worth(i) : 0u;
        const unsigned same = __ballot_sync(0xffffffffu, i < n && x == prefix);
        const bool stays = i < n && (x > prefix || (x == prefix && before + __popc(same & ((1u << lane) - 1u)) < wanted));
        const unsigned word = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) bits[w] = word;
        before += __popc(same);
    }
    __syncthreads();
    // numbers of the holes and of those that fill them
    const int per = (words + EV_THREADS - 1) / EV_THREADS;
    const int a0 = min(words, tid * per), a1 = min(words, a0 + per);
    auto below = [&](int w) -> unsigned {                // the word's places below the budget
        const int m = budget - w * 32;
        return m <= 0 ? 0u : m >= 32 ? 0xffffffffu : (1u << m) - 1u;
    };
    unsigned holes = 0, fillers = 0;
    for (int w = a0; w < a1; ++w) {
        holes += __popc(~bits[w] & below(w));
        fillers += __popc(bits[w] & ~below(w));
    }
    unsigned hs = holes, fs = fillers;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, hs, o), y = __shfl_up_sync(0xffffffffu, fs, o);
        if (lane >= o) {
            hs += x;
            fs += y;
        }
    }
    if (lane == 31) {
        warp_s[warp][0] = hs;
        warp_s[warp][1] = fs;
    }
    __syncthreads();
    hs -= holes;
    fs -= fillers;
    unsigned moves = 0;
    for (int w = 0; w < EV_WARPS; ++w) {
        if (w < warp) {
            hs += warp_s[w][0];
            fs += warp_s[w][1];
        }
        moves += warp_s[w][0];
    }
    if (apart)
        for (int i = tid; i < budget; i += EV_THREADS) {
            if (!((bits[i >> 5] >> (i & 31)) & 1u)) continue;
            const int slot = slot_of(table, p.page_size, p.num_slots, i);
            if (slot < 0) continue;
            p.mass_out[plane + slot] = p.mass[plane + slot];
            p.positions_out[plane + slot] = p.positions[plane + slot];
        }
    for (unsigned m0 = 0; m0 < moves; m0 += EV_LIST) {
        const unsigned count = min((unsigned)EV_LIST, moves - m0);
        unsigned hr = hs, fr = fs;
        for (int w = a0; w < a1; ++w) {
            for (unsigned x = ~bits[w] & below(w); x; x &= x - 1, ++hr)
                if (hr - m0 < count) list_s[0][hr - m0] = slot_of(table, p.page_size, p.num_slots, w * 32 + __ffs(x) - 1);
            for (unsigned x = bits[w] & ~below(w); x; x &= x - 1, ++fr)
                if (fr - m0 < count) list_s[1][fr - m0] = slot_of(table, p.page_size, p.num_slots, w * 32 + __ffs(x) - 1);
        }
        __syncthreads();
        move_rows<U>(p, plane, layer, h, list_s, 0, count);
        __syncthreads();
    }
    before_next();
}

// The widest unit that divides a row's bytes and every address that rows begin at.
int unit_bytes(const void* k, const void* v, long long row_bytes) {
    const uintptr_t all = (uintptr_t)k | (uintptr_t)v | (uintptr_t)row_bytes;
    return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

template <typename U> int launch_commit(const CommitParams& p, cudaStream_t stream) {
    llb_launch(tree_commit_kernel<U>, dim3(p.S, llb_ceil_div(p.L, p.layers_a_block)), dim3(COMMIT_THREADS), 0, stream, p);
    return llb_check_launch("tree_commit");
}
template <typename U> int launch_evict(EvictParams p, int L, cudaStream_t stream) {
    const int places = p.max_pages * p.page_size, bit_words = (places + 31) / 32;
    // 32 places a thread leave an SM one block, which pays while there are no more triples than SMs (us, 16,000 places thinned to 1,024, heads
    // of 128: 20 triples 57, shared 42, the general kernel 62; 560 triples 341, the general kernel 220)
    if (places <= 8 * EV_THREADS || (places <= 32 * EV_THREADS && (long long)p.S * p.Hkv * L <= llb_device_sms())) {
        // Where there are fewer (layer, request, kv head) triples than SMs, the blocks of a cluster share a triple's moves (each finds all of them:
        // trips that all have to make anyway).  us with one block | shared: 4,001 places thinned to 1,024, heads of 128: 20 triples 31 | 18;
        // heads of 64: 2 triples 22 | 13, 48 triples 23 | 18; 16,000 places to 8,000: 20 triples 155 | 74.  One key of each goes: 5.3 | 5.3.
        // (Up to three blocks an SM: 48 triples 18 -> 22, 80 of 128 33 -> 29, one key 5.4 -> 7.4.)
        const long long blocks = (long long)p.S * p.Hkv * L;
        while (p.parts < 8 && 2 * p.parts * blocks <= llb_device_sms()) p.parts *= 2;
        const bool few = places <= 8 * EV_THREADS;
        auto kernel = p.parts > 1 ? (few ? cache_evict_kernel<U, 8, true> : cache_evict_kernel<U, 32, true>)
                                  : (few ? cache_evict_kernel<U, 8, false> : cache_evict_kernel<U, 32, false>);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(p.S * p.Hkv * p.parts, L);
        cfg.blockDim = dim3(EV_THREADS);
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = p.parts;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = p.parts > 1 ? 2 : 1;
        cudaLaunchKernelEx(&cfg, kernel, p);          // (a failure is the runtime's last error, which llb_check_launch reads)
        return llb_check_launch("cache_evict");
    }
    // two blocks an SM have room for 20,000 worths each; places beyond that are read again in every pass
    p.cache_places = places < 20000 ? places : 20000;
    if (bit_words > 8192) p.cache_places = 8192;
    const size_t smem = sizeof(unsigned) * ((size_t)bit_words + p.cache_places);
    static LlbSharedMemory room;
    cudaError_t e = room.allow(cache_evict_any_kernel<U>, smem);
    if (e != cudaSuccess) return llb_fail("cache_evict: cannot opt in to %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    llb_launch(cache_evict_any_kernel<U>, dim3(p.S * p.Hkv, L), dim3(EV_THREADS), smem, stream, p);
    return llb_check_launch("cache_evict");
}

}  // namespace

LLB_EXPORT int llb_tree_commit(const LlbTreeCommit* c, cudaStream_t stream) {
    if (c->S == 0) return 0;
    LLB_REQUIRE(c->S > 0 && c->T >= 0 && c->L > 0 && c->L <= 65535 && c->max_pages >= 0 && c->page_size > 0 && c->num_slots > 0 && c->row_bytes > 0 &&
                c->row_bytes % 2 == 0 && (long long)c->max_pages * c->page_size <= (1 << 30), "tree_commit: bad sizes");
    LLB_REQUIRE(c->width > 0 && c->width <= COMMIT_MAX_PATH, "tree_commit: path has room for %d nodes, 1 to %d are possible", c->width, COMMIT_MAX_PATH);
    const long long rows = 4ll * c->T, spans = 4ll * c->S, planes = (long long)c->L * c->num_slots * c->row_bytes;
    if (int rc = llb_refuse_overlap("tree_commit", {{"k_cache", c->k, planes}, {"v_cache", c->v, planes}, {"path", c->path, spans * c->width},
                                                    {"count", c->count, spans}, {"next_token", c->next, spans}},
                                    {{"tokens", c->tokens, rows}, {"parents", c->parents, rows}, {"targets", c->targets, rows},
                                     {"span_row", c->span_row, spans}, {"span_len", c->span_len, spans}, {"span_pos", c->span_pos, spans},
                                     {"block_table", c->table, spans * c->max_pages}}))
        return rc;
    CommitParams p;
    p.tokens = c->tokens; p.parents = c->parents; p.targets = c->targets; p.k = (char*)c->k; p.v = (char*)c->v; p.span_row = c->span_row;
    p.span_len = c->span_len; p.span_pos = c->span_pos; p.table = c->table; p.S = c->S; p.T = c->T; p.L = c->L; p.max_pages = c->max_pages;
    p.page_size = c->page_size; p.num_slots = c->num_slots; p.path = c->path; p.width = c->width; p.count = c->count; p.next = c->next;
    const int unit = unit_bytes(c->k, c->v, c->row_bytes);
    p.row_units = c->row_bytes / unit;
    p.layers_a_block = COMMIT_THREADS / (2 * p.row_units) > 1 ? COMMIT_THREADS / (2 * p.row_units) : 1;
    if (unit == 16) return launch_commit<uint4>(p, stream);
    if (unit == 8) return launch_commit<uint2>(p, stream);
    if (unit == 4) return launch_commit<unsigned>(p, stream);
    return launch_commit<unsigned short>(p, stream);
}

LLB_EXPORT int llb_cache_evict(const LlbCacheEvict* c, cudaStream_t stream) {
    if (c->S == 0) return 0;
    LLB_REQUIRE(c->S > 0 && c->L > 0 && c->L <= 65535 && c->Hkv > 0 && (long long)c->S * c->Hkv < (1ll << 31) && c->page_size > 0 && c->max_pages >= 0 &&
                c->num_slots > 0 && c->head_bytes > 0 && c->head_bytes % 2 == 0, "cache_evict: bad sizes");
    LLB_REQUIRE((long long)c->max_pages * c->page_size <= EV_MAX_PLACES, "cache_evict: a block table of %d pages of %d names more than %d places",
                c->max_pages, c->page_size, EV_MAX_PLACES);
    LLB_REQUIRE(c->budget > 0 && c->first >= 0 && c->latest >= 0 && (long long)c->first + c->latest <= c->budget,
                "cache_evict: a budget of %d places does not hold the first %d and the latest %d", c->budget, c->first, c->latest);
    const long long spans = 4ll * c->S, heads = (long long)c->L * c->Hkv * c->num_slots, planes = heads * c->head_bytes;
    const bool apart = c->mass_out != c->mass || c->positions_out != c->positions;
    if (int rc = llb_refuse_overlap("cache_evict", {{"k_cache", c->k, planes}, {"v_cache", c->v, planes}, {"mass_out", c->mass_out, 4 * heads},
                                                    {"positions_out", c->positions_out, 4 * heads}},
                                    {{"mass", apart ? c->mass : nullptr, 4 * heads}, {"positions", apart ? c->positions : nullptr, 4 * heads},
                                     {"lengths", c->lengths, spans}, {"ends", c->ends, spans}, {"block_table", c->table, spans * c->max_pages}}))
        return rc;
    EvictParams p;
    p.k = (char*)c->k; p.v = (char*)c->v; p.mass = c->mass; p.positions = c->positions; p.mass_out = c->mass_out; p.positions_out = c->positions_out;
    p.lengths = c->lengths; p.ends = c->ends; p.table = c->table; p.S = c->S; p.max_pages = c->max_pages; p.page_size = c->page_size;
    p.num_slots = c->num_slots; p.Hkv = c->Hkv; p.budget = c->budget; p.first = c->first; p.latest = c->latest; p.cache_places = 0; p.parts = 1;
    const int unit = unit_bytes(c->k, c->v, c->head_bytes);
    p.head_units = c->head_bytes / unit;
    if (unit == 16) return launch_evict<uint4>(p, c->L, stream);
    if (unit == 8) return launch_evict<uint2>(p, c->L, stream);
    if (unit == 4) return launch_evict<unsigned>(p, c->L, stream);
    return launch_evict<unsigned short>(p, c->L, stream);
}
