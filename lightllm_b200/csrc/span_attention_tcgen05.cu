// Attention over whole requests on the 5th-generation tensor cores (sm_100a, bf16, heads of 64 and 128): rows with a tree mask or causal
// ones, and the sums of the weights that keys receive.  Which rows see which keys, jobs and their cut: span_attention.cuh.
//
// 128 (row, head of the group) pairs are the 128 lanes of tensor memory, so all query heads that read the same keys read them at
// once: a few drafted nodes fill the lanes that their heads' keys pay for anyway.  A block has two softmax groups of 128 threads (a
// thread a lane) and one line of key tiles that are loaded once:
//     more than 128 pairs     each group has 128 pairs of its own, both see every tile
//     up to 128 pairs         both have the same pairs, the first sees the even tiles and the second the odd ones; they are joined at
//                             the end through tensor memory (the same pair has the same lane in both)
// While one group works on its scores the tensor cores work for the other.  (Strict turns at the exponentials were built: a pair of tiles took
// 4,200 cycles instead of 3,600.)  For every tile of 128 keys of a group:
//     S = Q K^T               tcgen05.mma, 128 columns of tensor memory, in two halves of 64 keys
//     m, p = 2^(S - m), l     a thread reads its lane's 128 scores once; p goes back to tensor memory as bf16 (over the second half of S)
//                             and is the A operand of the next product without a way through shared memory
//                             (bf16 because both operands of a product have the type of V: a weight is off by half a step, 2^-8 of it, and
//                             the sum l is taken before that rounding.  Against 64 bits results are up to 4 % further off than with P in 32
//                             bits, 1.73e-3 instead of 1.67e-3: their own rounding to bf16 is most of it.  2^x is ex2.approx, off by 2^-22)
//     O += P V                in tensor memory; it is scaled only when a lane's maximum has grown by more than 2^8 since its last
//                             scaling (any reference works for a softmax, and 2^8 leaves floats and bf16 their accuracy)
// K and V tiles go through a ring of half tiles (128 keys of K, or of V) that TMA fills page by page, several ahead, across jobs.
#include <cuda.h>

#include "span_attention.cuh"
#include "tcgen05_common.cuh"
#include "warp_mma.cuh"

namespace {

using namespace t5;
using wm::fast_exp2;

constexpr int BQ = 128, BK = 128;
constexpr int NUM_THREADS = 384;               // two softmax groups of 128; a third with the warp that issues products and the loader warp
constexpr int MMA_WARP = 8, LOAD_WARP = 9;
constexpr uint32_t TILE_BYTES = 128 * 128;     // [128 rows][64 elements]
constexpr float RESCALE = 8.0f;                // how far (powers of two) a lane's maximum may pass its reference
constexpr int BAR_PAIR = 1;                    // both softmax groups; 2 and 3: each of them

template <int HD> struct Shape {
    static constexpr int KB = HD / 64;
    static constexpr uint32_t HALF = KB * TILE_BYTES;           // 128 rows of Q, K or V
    static constexpr int RING = HD == 64 ? 10 : 5;
    static constexpr size_t SMEM = (size_t)(2 + RING) * HALF + 1024;
};

struct TcParams {
    LlbSpanArgs a;
    const __nv_bfloat16* v;
    int pairs_nodes;            // rows of a request whose pairs fill 128 lanes
    int* error_flag;
};

// A block is launched with 3 x 168 registers a thread of its three groups; the third one needs few, the softmax groups hold a row
// of 128 scores: 104 + 2 x 200 = 504.
__device__ __forceinline__ void registers_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 104;"); }
__device__ __forceinline__ void registers_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 200;"); }
__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
// One lane of the warp, chosen by the hardware's own election: the compiler then knows that a single lane runs what follows, and keeps
// descriptors and addresses in the uniform registers that a product takes.  Under `lane == 0` it brings each of them there first, and
// beside eight busy warps a 128 x 128 x 16 product costs the issuing one 83 to 350 cycles instead of 65 (64 is the tensor cores' own time).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
// D[128 x N] += A B with A in tensor memory (bf16, two to a column).
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
        ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
}
// A 128 x N tile of scores, both operands K-major in shared memory.
template <int KB> __device__ __forceinline__ void issue_scores(uint32_t tmem, uint32_t a_addr, uint32_t b_addr, uint32_t idesc) {
    const uint64_t da = desc_kmajor(a_addr), db = desc_kmajor(b_addr);
    umma_bf16_first(tmem, da, db, idesc);
#pragma unroll
    for (int k = 1; k < 4 * KB; ++k) {
        const uint64_t step = (k >> 2) * (TILE_BYTES >> 4) + (k & 3) * 2;
        umma_bf16_acc(tmem, da + step, db + step, idesc);
    }
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&u)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
          "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
          "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]),
          "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
        : "memory");
}
// The loads before this have completed; what uses their 32 registers stays behind it.
__device__ __forceinline__ void tmem_wait_ld32(float (&r)[32]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]),
                   "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]),
                   "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]),
                   "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// What the loader has asked for arrives before its block ends, whoever gave up on a wait: of every barrier that loads complete on, the last of
// the `loads` that it had (they take turns: a barrier has one at a time).  With a limit, as every wait.
__device__ __forceinline__ void loads_arrive(uint64_t* bar, uint32_t loads) {
    if (loads == 0) return;
    const long long since = clock64();
    while (!mbar_try_wait(bar, (loads - 1) & 1) && clock64() - since < WAIT_LIMIT_CYCLES / 64) {
    }
}
// Of those that `loaded` loads went through one after the other.
template <int RING> __device__ __forceinline__ void ring_arrives(uint64_t (&bar)[RING], uint32_t loaded) {
    for (uint32_t i = 0; i < RING; ++i) loads_arrive(&bar[i], (loaded + RING - 1 - i) / RING);
}

// A row's mask.  The first two words (128 nodes) are asked for when the job begins, since a trip to memory in the last tile would be as long as
// the rest of its work.
struct RowMask {
    const unsigned long long* row;
    int words;
    unsigned long long w0, w1;
    __device__ __forceinline__ unsigned long long word(int w) const { return w == 0 ? w0 : w == 1 ? w1 : w < words ? row[w] : 0ull; }
    // 32 bits from node j0 on (which may be negative), those of nodes from len on cleared
    __device__ __forceinline__ uint32_t bits(int j0, int len) const {
        if (j0 <= -32 || j0 >= len) return 0u;
        uint32_t x;
        if (j0 < 0) x = (uint32_t)w0 << -j0;
        else {
            const int w = j0 >> 6, sh = j0 & 63;
            unsigned long long y = word(w) >> sh;
            if (sh > 32) y |= word(w + 1) << (64 - sh);
            x = (uint32_t)y;
        }
        return len - j0 < 32 ? x & ((1u << (len - j0)) - 1u) : x;
    }
};
__device__ __forceinline__ uint32_t first_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ bool bf16_odd(uint32_t pair) { return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u; }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The largest of a lane's 128 scores.
__device__ __forceinline__ float tile_max(uint32_t tmem) {
    float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 128; c += 32) {
        float s[32];
        tmem_ld32(tmem + c, s);
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            t0 = max3(t0, s[i], s[i + 1]);
            t1 = max3(t1, s[i + 2], s[i + 3]);
            t2 = max3(t2, s[i + 4], s[i + 5]);
            t3 = max3(t3, s[i + 6], s[i + 7]);
        }
    }
    return fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
}
// 2^(score * scale + shift) of a lane's 128 scores as bf16 pairs, their sum (before the rounding) and the largest score, which tells
// whether the shift was near enough: after the first tile it nearly always is, so that no pass for the maximum comes before this one.  The scores
// stay where they are.  second_half() is called when the second 64 of them are wanted.
template <typename SecondHalf>
__device__ __forceinline__ void tile_probs(uint32_t tmem, float scale, float shift, uint32_t (&probs)[64], float& sum, float& top,
                                           const SecondHalf& second_half) {
    float t0 = -INFINITY, t1 = -INFINITY;
    unsigned long long l0 = 0, l1 = 0;          // (sums two by two: the schedulers' slots are shared with the warp that issues the products)
    const unsigned long long scale2 = llb_pack2(scale, scale), shift2 = llb_pack2(shift, shift);
    float s[2][32];
    tmem_ld32_nowait(tmem, *reinterpret_cast<uint32_t(*)[32]>(&s[0][0]));
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        tmem_wait_ld32(s[c & 1]);
        if (c == 1) {
            second_half();
            __syncwarp();
        }
        if (c < 3) tmem_ld32_nowait(tmem + 32 * (c + 1), *reinterpret_cast<uint32_t(*)[32]>(&s[(c + 1) & 1][0]));
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float* v = &s[c & 1][i];
            t0 = max3(t0, v[0], v[1]);
            t1 = max3(t1, v[2], v[3]);
            float p0, p1, p2, p3;
            llb_unpack2(llb_fma2(llb_pack2(v[0], v[1]), scale2, shift2), p0, p1);
            llb_unpack2(llb_fma2(llb_pack2(v[2], v[3]), scale2, shift2), p2, p3);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            p2 = fast_exp2(p2);
            p3 = fast_exp2(p3);
            l0 = llb_add2(l0, llb_pack2(p0, p1));
            l1 = llb_add2(l1, llb_pack2(p2, p3));
            probs[16 * c + i / 2] = wm::pack_bf16(p0, p1);
            probs[16 * c + i / 2 + 1] = wm::pack_bf16(p2, p3);
        }
    }
    float a, b;
    llb_unpack2(llb_add2(l0, l1), a, b);
    sum = a + b;
    top = fmaxf(t0, t1);
}

// Four bytes a page: the cache row that a page of a tile begins at, or num_slots (TMA reads zeros there) for one that holds no key of
// the job or is none of the cache's.
__device__ __forceinline__ int page_row(const LlbSpanArgs& a, int s, int page_of, int keys) {
    if (page_of >= a.max_pages || page_of * a.page_size >= keys) return a.num_slots;
    const int page = a.table[(size_t)s * a.max_pages + page_of];
    return page >= 0 && (long long)page * a.page_size < a.num_slots ? page * a.page_size : a.num_slots;
}

// What the roles share of a block's walk through its jobs.
struct Segment {
    int k0, k1;              // tiles of the job
    bool two;                // the groups have pairs of their own
    int part;
};
__device__ __forceinline__ Segment segment_of(const TcParams& p, const LlbPiece& pc, const LlbJob& job, int t) {
    Segment g;
    g.k0 = t - job.begin;
    g.k1 = min(job.tiles, pc.t1 - job.begin);
    g.two = job.count(p.a) > p.pairs_nodes;
    g.part = llb_part_of(pc, job);
    return g;
}

// On to the next job, if the piece goes on.
__device__ __forceinline__ bool next_job(const LlbSpanArgs& a, const LlbPiece& pc, LlbJob& job, int& t) {
    t = job.begin + job.tiles + a.extra;
    if (t >= pc.t1) return false;
    job.next(a, BK);
    return true;
}

template <int HD>
__global__ void __launch_bounds__(NUM_THREADS, 1)
span_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const TcParams p) {
    constexpr int KB = Shape<HD>::KB, RING = Shape<HD>::RING;
    constexpr uint32_t HALF = Shape<HD>::HALF;
    constexpr uint32_t TMEM_COLS = 512;              // S (and P) of the groups: 0.., 128..; O: 256.., 384..
    __shared__ __align__(8) uint64_t bar_q_full[2], bar_q_free[2], bar_kv_full[RING], bar_kv_free[RING], bar_s[4], bar_p[2], bar_o[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s, odd_s;
    __shared__ LlbPiece piece_s;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = smem;                             // two buffers
    uint8_t* ring = smem + 2 * HALF;
    volatile int* abort_flag = &abort_s;
    const LlbSpanArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_q_full[i], 1);
            mbar_init(&bar_q_free[i], 1);
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_s[2 + i], 1);
            mbar_init(&bar_p[i], 4);
            mbar_init(&bar_o[i], 1);
        }
        for (int i = 0; i < RING; ++i) {
            mbar_init(&bar_kv_full[i], 1);
            mbar_init(&bar_kv_free[i], 2);
        }
        abort_s = 0;
        odd_s = 0;
        mbar_init_fence();
    }
    if (warp == MMA_WARP) tmem_alloc(&tmem_slot, TMEM_COLS);
    griddep_wait();
    griddep_launch_dependents();
    if (warp == 0) {
        const LlbPiece pc = llb_piece(a, BK, blockIdx.x, gridDim.x, LLB_SPAN_TC_LEAST, lane);
        if (lane == 0) {
            piece_s = pc;
            llb_leave_open(a, pc, pc.job, false);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    const LlbPiece pc = piece_s;
    LlbJob job = pc.job;
    constexpr uint32_t IDESC_S = idesc_bf16(BQ, BK / 2, 0), IDESC_PV = idesc_bf16(BQ, HD, 1);
    // Q buffers: jobs of two pair tiles take both, others one after the other
    int q_next = 0;
    uint32_t tiles_before = 0;                       // tiles of the block's jobs before this one

    if (warp >= MMA_WARP) {
    registers_give();
    if (warp == LOAD_WARP) {
        bool ok = true;
        const uint32_t q_bytes = (uint32_t)p.pairs_nodes * a.group * 128 * KB;
        const int ppt = BK / a.page_size;
        uint32_t loaded = 0, q_phases = 0;           // of bar_q_free (bits 0, 1), and which buffers have been used (bits 2, 3)
        uint32_t q_loaded[2] = {0, 0};
#pragma unroll 1
        for (int t = pc.t0; t < pc.t1;) {
            const Segment g = segment_of(p, pc, job, t);
            if (g.k0 >= job.tiles) {
                if (!next_job(a, pc, job, t)) break;
                continue;
            }
#pragma unroll 1
            for (int x = 0; x < (g.two ? 2 : 1); ++x) {
                const int b = g.two ? x : q_next;
                if ((q_phases >> (2 + b)) & 1) {
                    ok = mbar_wait(&bar_q_free[b], (q_phases >> b) & 1, abort_flag) && ok;
                    q_phases ^= 1u << b;
                }
                q_phases |= 4u << b;
                if (ok) {
                    if (lane == 0) {
                        mbar_expect_tx(&bar_q_full[b], q_bytes);
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb)
                            tma_load_3d(q_s + b * HALF + kb * TILE_BYTES, &map_q, kb * 64, job.kvh * a.group,
                                        job.z.row + job.first + x * p.pairs_nodes, &bar_q_full[b]);
                    }
                    ++(b == 0 ? q_loaded[0] : q_loaded[1]);
                }
            }
            if (!g.two) q_next ^= 1;
#pragma unroll 1
            for (int k = g.k0; k < g.k1; ++k) {
                const int row = lane < ppt ? page_row(a, job.s, k * ppt + lane, job.keys) : a.num_slots;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t slot = loaded % RING;
                    if (loaded >= RING) ok = mbar_wait(&bar_kv_free[slot], (loaded / RING - 1) & 1, abort_flag) && ok;
                    if (ok) {
                        if (lane == 0) mbar_expect_tx(&bar_kv_full[slot], HALF);
                        __syncwarp();
                        if (lane < ppt) {
                            uint8_t* dst = ring + slot * HALF + (uint32_t)lane * a.page_size * 128;
#pragma unroll
                            for (int kb = 0; kb < KB; ++kb)
                                tma_load_2d(dst + kb * TILE_BYTES, half ? &map_v : &map_k, job.kvh * HD + kb * 64, row, &bar_kv_full[slot]);
                        }
                        ++loaded;
                    }
                    __syncwarp();
                }
            }
            if (!next_job(a, pc, job, t)) break;
        }
        ring_arrives(bar_kv_full, loaded);
        loads_arrive(&bar_q_full[0], q_loaded[0]);
        loads_arrive(&bar_q_full[1], q_loaded[1]);
    } else if (warp == MMA_WARP && elect_one()) {
        bool ok = true;
        uint32_t phases = 0;                         // the next phase of bar_p (bits 0, 1) and bar_q_full (bits 2, 3)
        auto full = [&](uint32_t half) {             // half tile number `half` of the block has arrived
            ok = mbar_wait(&bar_kv_full[half % RING], (half / RING) & 1, abort_flag) && ok;
            tc_fence_after();
        };
        // The scores come in two halves: the first one of the next tile goes ahead of this tile's P V, so that the softmax goes on with it
        // meanwhile; the second one, which takes the place of P, follows it.
        auto issue_s = [&](int x, int b, uint32_t half, int which) {
            if (!ok) return;
            issue_scores<KB>(tmem_base + x * 128 + which * 64, smem_u32(q_s + b * HALF), smem_u32(ring + half % RING * HALF) + which * 64 * 128, IDESC_S);
            umma_commit(&bar_s[2 * which + x]);
        };
#pragma unroll 1
        for (int t = pc.t0; t < pc.t1;) {
            const Segment g = segment_of(p, pc, job, t);
            if (g.k0 >= job.tiles) {
                if (!next_job(a, pc, job, t)) break;
                continue;
            }
            const int n = g.k1 - g.k0, step = g.two ? 1 : 2;
            const int buf0 = g.two ? 0 : q_next, buf1 = g.two ? 1 : q_next;
#pragma unroll 1
            for (int x = 0; x < 2; ++x) {
                const int b = x == 0 ? buf0 : buf1;
                if (g.two || x == 0) {
                    ok = mbar_wait(&bar_q_full[b], (phases >> (2 + b)) & 1, abort_flag) && ok;
                    phases ^= 4u << b;
                }
                const int first = g.two ? 0 : x;
                if (first >= n) continue;
                full(2 * (tiles_before + first));
                issue_s(x, b, 2 * (tiles_before + first), 0);
                issue_s(x, b, 2 * (tiles_before + first), 1);
            }
            if (!g.two) q_next ^= 1;
#pragma unroll 1
            for (int j0 = 0; j0 < n; j0 += step) {
#pragma unroll 1
                for (int x = 0; x < 2; ++x) {
                    const int j = g.two ? j0 : j0 + x;
                    if (j >= n) continue;
                    const uint32_t half = 2 * (tiles_before + j);
                    const bool more = j + step < n;
                    if (more) full(half + 2 * step);
                    ok = mbar_wait(&bar_p[x], (phases >> x) & 1, abort_flag) && ok;
                    phases ^= 1u << x;
                    tc_fence_after();
                    if (more) issue_s(x, x == 0 ? buf0 : buf1, half + 2 * step, 0);
                    full(half + 1);
                    if (ok) {
                        const uint64_t dv = desc_mnmajor(smem_u32(ring + (half + 1) % RING * HALF), TILE_BYTES);
                        const uint32_t to = tmem_base + 256 + x * 128, from = tmem_base + x * 128 + 64;
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            umma_ts(to, from + k * 8, dv + k * (16 * 128 >> 4), IDESC_PV, (j0 > 0 || k > 0) ? 1u : 0u);
                    }
                    if (more) issue_s(x, x == 0 ? buf0 : buf1, half + 2 * step, 1);          // (its commit is behind P V, too)
                    else if (ok) umma_commit(&bar_o[x]);
                }
            }
            tiles_before += n;
            if (!next_job(a, pc, job, t)) break;
        }
    }
    } else {
        registers_take();
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem_base + x * 128 + lanes, tmem_o = tmem_base + 256 + lanes;
        bool ok = true;
        uint32_t n_s = 0, n_o = 0;
#pragma unroll 1
        for (int t = pc.t0; t < pc.t1;) {
            const Segment g = segment_of(p, pc, job, t);
            if (g.k0 >= job.tiles) {
                if (!next_job(a, pc, job, t)) break;
                continue;
            }
            const int n = g.k1 - g.k0, step = g.two ? 1 : 2;
            const int node0 = g.two ? x * p.pairs_nodes : 0;
            const int pairs = min(p.pairs_nodes, job.count(a) - node0) * a.group;
            const bool mine = r < pairs;
            const int node = job.first + node0 + (mine ? r / a.group : 0);
            const LlbSpan z = job.z;
            const unsigned long long* mask = a.mask ? a.mask + (size_t)(z.row + node) * a.words : nullptr;
            const RowMask row_mask = {mask, a.words, mask && mine ? mask[0] : 0ull, mask && mine && a.words > 1 ? mask[1] : 0ull};
            const int all = a.mask ? z.pos : z.pos + job.first + 1;         // keys that every row of the job sees
            const int own = a.mask ? z.pos : z.pos + node + 1;              // first keys that this row sees
            const bool busy = (warp & 3) * 32 < pairs;                      // any pair in this warp's lanes
            float m_ref = -INFINITY, l_run = mine ? llb_first_sum(a, z, node) : 0.0f;
#pragma unroll 1
            for (int j = g.two ? 0 : x; j < n; j += step) {
                const int key0 = (g.k0 + j) * BK;
                const uint32_t half = 2 * (tiles_before + j);
                ok = mbar_wait(&bar_s[x], n_s & 1, abort_flag) && ok;
                tc_fence_after();
                // The second half of S: it has read K, and the product before it V; Q, if this is the job's last tile.
                bool whole = false;
                auto second_half = [&]() {
                    if (whole) return;
                    whole = true;
                    ok = mbar_wait(&bar_s[2 + x], n_s & 1, abort_flag) && ok;
                    tc_fence_after();
                    if (r == 0) {
                        mbar_arrive_n(&bar_kv_free[half % RING], g.two ? 1 : 2);
                        if (j >= step) mbar_arrive_n(&bar_kv_free[(half + 1 - 2 * step) % RING], g.two ? 1 : 2);
                        if (g.two && j + 1 == n) mbar_arrive(&bar_q_free[x]);
                    }
                };
                const bool interior = key0 + BK <= all;
                if (!interior || j < step || a.scores || !busy) second_half();
                if (!interior) {
                    // Values that no row or not every row sees: what earlier owners left behind the last key, and numbers that are
                    // none in rows that see them, would reach the other rows as 0 * inf.  They become zeros here; rows that see the
                    // latter get them back at the end.
                    ok = mbar_wait(&bar_kv_full[(half + 1) % RING], ((half + 1) / RING) & 1, abort_flag) && ok;
                    const int key = key0 + r;
                    if (key >= all && ok) {
                        uint8_t* row = ring + (half + 1) % RING * HALF + (uint32_t)r * 128;
#pragma unroll 1
                        for (int kb = 0; kb < KB; ++kb)
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                // (neighbouring threads begin at other chunks: their rows lie in the same banks)
                                uint4* at = reinterpret_cast<uint4*>(row + kb * TILE_BYTES + ((c ^ r) & 7) * 16);
                                if (key >= job.keys) {
                                    *at = make_uint4(0u, 0u, 0u, 0u);
                                    continue;
                                }
                                uint4 w = *at;
                                if (bf16_odd(w.x) || bf16_odd(w.y) || bf16_odd(w.z) || bf16_odd(w.w)) {
                                    odd_s = 1;
                                    __threadfence_block();
                                    uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        if ((u[e] & 0x7f80u) == 0x7f80u) u[e] &= 0xffff0000u;
                                        if ((u[e] & 0x7f800000u) == 0x7f800000u) u[e] &= 0xffffu;
                                    }
                                    *at = w;
                                }
                            }
                    }
                    fence_async_smem();
                }
                if (busy) {
                    if (!interior) {
                        // what this row does not see becomes minus infinity where it stands
#pragma unroll 1
                        for (int w = 0; w < 4; ++w) {
                            uint32_t bits = first_bits(own - key0 - 32 * w);
                            if (mask && mine) bits |= row_mask.bits(key0 + 32 * w - z.pos, z.len);
                            __syncwarp();
                            float s[32];
                            tmem_ld32(tmem_s + 32 * w, s);
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[i] = (bits >> i) & 1u ? s[i] : -INFINITY;
                            tmem_st32(tmem_s + 32 * w, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
                        }
                        tmem_wait_st();
                    }
                    if (a.scores && z.len == 1 && job.begin + g.k0 + j < a.score_tiles) {
                        float* to = a.scores + ((size_t)(job.begin + g.k0 + j) * a.group + r) * BK;
#pragma unroll 1
                        for (int c = 0; c < 128; c += 32) {
                            float s[32];
                            __syncwarp();
                            tmem_ld32(tmem_s + c, s);
                            if (mine) {
#pragma unroll
                                for (int i = 0; i < 32; i += 4)
                                    *reinterpret_cast<float4*>(to + c + i) = make_float4(s[i] * a.scale_log2e, s[i + 1] * a.scale_log2e,
                                                                                         s[i + 2] * a.scale_log2e, s[i + 3] * a.scale_log2e);
                            }
                        }
                        __syncwarp();
                    }
                    if (j < step) m_ref = tile_max(tmem_s) * a.scale_log2e;              // (no O yet)
                    uint32_t probs[64];
                    float sum, top;
                    tile_probs(tmem_s, a.scale_log2e, m_ref == -INFINITY ? 0.0f : -m_ref, probs, sum, top, second_half);
                    top *= a.scale_log2e;
                    if (__any_sync(0xffffffffu, top > m_ref + RESCALE)) {
                        float corr = 1.0f;
                        if (top > m_ref + RESCALE) {
                            corr = m_ref == -INFINITY ? 0.0f : fast_exp2(m_ref - top);
                            m_ref = top;
                        }
                        l_run *= corr;
                        __syncwarp();
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            float o[32];
                            tmem_ld32(tmem_o + x * 128 + c, o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= corr;
                            tmem_st32(tmem_o + x * 128 + c, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
                        }
                        tile_probs(tmem_s, a.scale_log2e, m_ref == -INFINITY ? 0.0f : -m_ref, probs, sum, top, second_half);
                    }
                    l_run += sum;
                    tmem_st32(tmem_s + 64, *reinterpret_cast<const uint32_t(*)[32]>(&probs[0]));
                    tmem_st32(tmem_s + 96, *reinterpret_cast<const uint32_t(*)[32]>(&probs[32]));
                    tmem_wait_st();
                }
                ++n_s;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_p[x]);
            }
            const bool any = g.two || x < n;
            if (any) {
                ok = mbar_wait(&bar_o[x], n_o++ & 1, abort_flag) && ok;
                tc_fence_after();
                if (r == 0) {
                    const int last = g.two ? n - 1 : x + (n - 1 - x) / 2 * 2;
                    mbar_arrive_n(&bar_kv_free[(2 * (tiles_before + last) + 1) % RING], g.two ? 1 : 2);
                }
            }
            const int buf = g.two ? x : q_next;
            float w_own = 1.0f, w_other = 0.0f;
            if (!g.two) {
                // the groups' maxima and sums meet in the job's Q buffer, which nothing reads any more once both have passed
                float2* meet = reinterpret_cast<float2*>(q_s + buf * HALF);
                named_barrier(BAR_PAIR, 256);
                meet[x * 128 + r] = make_float2(m_ref, l_run);
                named_barrier(BAR_PAIR, 256);
                const float2 other = meet[(x ^ 1) * 128 + r];
                const float M = fmaxf(m_ref, other.x);
                w_own = m_ref == -INFINITY ? (l_run == 0.0f ? 0.0f : 1.0f) : fast_exp2(m_ref - M);
                w_other = other.x == -INFINITY ? (other.y == 0.0f ? 0.0f : 1.0f) : fast_exp2(other.x - M);
                l_run = l_run * w_own + other.y * w_other;
                m_ref = M;
                q_next ^= 1;
            }
            const int head = job.kvh * a.group + (mine ? r % a.group : 0), row = z.row + node;
            const int d0 = g.two ? 0 : x * (HD / 2), d1 = g.two ? HD : d0 + HD / 2;
            const float inv = 1.0f / l_run;
            const bool both = !g.two && n > 1;
            const bool odd = *(volatile int*)&odd_s != 0;
            if (busy) {
#pragma unroll 1
                for (int c = d0; c < d1; c += 32) {
                    float o[32];
                    __syncwarp();
                    if (g.two) {
                        tmem_ld32(tmem_o + x * 128 + c, o);
                    } else {
                        // (group 0 has tiles in any case)
                        tmem_ld32(tmem_o + c, o);
                        const float w0 = x == 0 ? w_own : w_other, w1 = x == 0 ? w_other : w_own;
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= w0;
                        if (both) {
                            float o1[32];
                            tmem_ld32(tmem_o + 128 + c, o1);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = fmaf(o1[i], w1, o[i]);
                        }
                    }
                    if (odd && mine) {
#pragma unroll 1
                        for (int key = max(all, g.k0 * BK); key < min(job.keys, g.k1 * BK); ++key) {
                            const int jn = key - z.pos;
                            const bool sees = mask ? (mask[jn >> 6] >> (jn & 63)) & 1ull : jn <= node;
                            const int slot = sees ? llb_span_slot(a, job.s, key) : -1;
                            if (slot < 0) continue;
                            const uint32_t* vr = reinterpret_cast<const uint32_t*>(p.v + ((size_t)slot * a.Hkv + job.kvh) * HD + c);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint32_t w = vr[i];
                                if ((w & 0x7f80u) == 0x7f80u) o[2 * i] += __uint_as_float(w << 16);
                                if ((w & 0x7f800000u) == 0x7f800000u) o[2 * i + 1] += __uint_as_float(w & 0xffff0000u);
                            }
                        }
                    }
                    if (!mine || !ok) {
                    } else if (g.part >= 0) {
                        float4* po = reinterpret_cast<float4*>(a.part_o) + ((size_t)(blockIdx.x * 2 + g.part) * (HD / 4) + c / 4) * a.rows + node0 * a.group + r;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) po[(size_t)(i / 4) * a.rows] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    } else {
                        __nv_bfloat16* dst = (__nv_bfloat16*)a.out + ((size_t)row * a.Hq + head) * HD + c;
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4*>(dst + i) =
                                make_uint4(wm::pack_bf16(o[i] * inv, o[i + 1] * inv), wm::pack_bf16(o[i + 2] * inv, o[i + 3] * inv),
                                           wm::pack_bf16(o[i + 4] * inv, o[i + 5] * inv), wm::pack_bf16(o[i + 6] * inv, o[i + 7] * inv));
                    }
                }
            }
            if (mine && ok && (g.two || x == 0)) {
                if (g.part >= 0) {
                    float* ml = a.part_ml + ((size_t)(blockIdx.x * 2 + g.part) * a.rows + node0 * a.group + r) * 2;
                    ml[0] = m_ref;
                    ml[1] = l_run;
                } else if (a.lse) {
                    a.lse[(size_t)row * a.Hq + head] = llb_lse(m_ref, l_run);
                }
            }
            if (g.part == 1 && threadIdx.x == 0) llb_leave_open(a, pc, job, true);
            // O is free for the next job, and Q where the groups met in it (they have read each other's O)
            tc_fence_before();
            fence_async_smem();
            if (!g.two) named_barrier(BAR_PAIR, 256);
            else named_barrier(BAR_PAIR + 1 + x, 128);
            if (!g.two && r == 0 && x == 0) mbar_arrive(&bar_q_free[buf]);
            tiles_before += n;
            if (!next_job(a, pc, job, t)) break;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 4);
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// ---- the weights that keys receive -----------------------------------------------------------------------------------------------
// mass_j = sum over rows i and heads of 2^(x_ij - lse_i), the scores made once more with keys and queries in each other's place:
//     S^T = K Q^T             128 keys are the lanes, 128 (row, head) pairs the columns
// so that a key's sum is a sum in one thread's register, made in one order, with no meeting of threads and no atomics.  What bounds it
// is the exponential of every score (16 a cycle and SM).  A job is a tile of 128 keys of one request and kv head; the tiles of rows
// that see any of its keys make the line that is cut among the blocks, as above; K stays in shared memory for the job, the tiles of Q
// go through the ring, every other one to one of two groups of 128 threads, each with two score tiles in tensor memory so that
// the next is made while one is read.
struct MassArgs {
    TcParams p;
    float* part;                // [2 * blocks, 128]
};

template <int HD> struct MassShape {
    static constexpr int RING = HD == 64 ? 8 : 4;
    static constexpr size_t SMEM = (size_t)(2 + RING) * Shape<HD>::HALF + 1024;
};

template <int HD>
__global__ void __launch_bounds__(NUM_THREADS, 1)
span_mass_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const MassArgs m) {
    constexpr int KB = Shape<HD>::KB, RING = MassShape<HD>::RING;
    constexpr uint32_t HALF = Shape<HD>::HALF;
    constexpr uint32_t TMEM_COLS = 512;              // two score tiles of each group
    __shared__ __align__(8) uint64_t bar_k_full[2], bar_k_free[2], bar_q_full[RING], bar_q_free[RING], bar_s[4], bar_free[4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s;
    __shared__ LlbMassPiece piece_s;
    __shared__ __align__(16) float lse_s[8][2][128];          // a warp's own, so that no group has to meet
    __shared__ float sum_s[128];
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* k_s = smem;                             // two buffers: this job's and the next one's
    uint8_t* ring = smem + 2 * HALF;
    volatile int* abort_flag = &abort_s;
    const LlbSpanArgs& a = m.p.a;
    const int pairs_nodes = m.p.pairs_nodes, pairs_tile = pairs_nodes * a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_k_full[i], 1);
            mbar_init(&bar_k_free[i], 1);
        }
        for (int i = 0; i < RING; ++i) {
            mbar_init(&bar_q_full[i], 1);
            mbar_init(&bar_q_free[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_free[i], 4);
        }
        abort_s = 0;
        mbar_init_fence();
    }
    if (warp == MMA_WARP) tmem_alloc(&tmem_slot, TMEM_COLS);
    // columns that no pair has (128 is no multiple of the group) stay zero
    for (int i = threadIdx.x; i < RING * KB * (128 - pairs_tile) * 8; i += NUM_THREADS) {
        const int tile = i / ((128 - pairs_tile) * 8), rest = i - tile * ((128 - pairs_tile) * 8);
        *reinterpret_cast<uint4*>(ring + (size_t)tile * TILE_BYTES + (pairs_tile + rest / 8) * 128 + rest % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_async_smem();
    griddep_wait();
    griddep_launch_dependents();
    if (warp == 0) {
        const LlbMassPiece pc = llb_mass_piece(a, BK, pairs_nodes, blockIdx.x, gridDim.x, lane);
        if (lane == 0) {
            piece_s = pc;
            llb_leave_open_mass(a, pc.line, pc.job, false);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    const LlbPiece pc = piece_s.line;
    LlbMassJob job = piece_s.job;
    uint32_t jobs = 0, units_before = 0;
    constexpr uint32_t IDESC = idesc_bf16(BK, BQ, 0);

    if (warp == LOAD_WARP) {
        bool ok = true;
        const uint32_t q_bytes = (uint32_t)pairs_tile * 128 * KB;
        const int ppt = BK / a.page_size;
        uint32_t loaded = 0, k_loaded = 0;
#pragma unroll 1
        for (int t = pc.t0; t < pc.t1;) {
            const int u0 = t - job.begin, u1 = min(job.units, pc.t1 - job.begin), b = jobs & 1;
            const int row = lane < ppt ? page_row(a, job.s, job.tile * ppt + lane, job.z.pos + job.z.len) : a.num_slots;
            if (jobs >= 2) ok = mbar_wait(&bar_k_free[b], (jobs / 2 - 1) & 1, abort_flag) && ok;
            if (ok) {
                if (lane == 0) mbar_expect_tx(&bar_k_full[b], HALF);
                __syncwarp();
                if (lane < ppt) {
                    uint8_t* dst = k_s + b * HALF + (uint32_t)lane * a.page_size * 128;
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) tma_load_2d(dst + kb * TILE_BYTES, &map_k, job.kvh * HD + kb * 64, row, &bar_k_full[b]);
                }
                ++k_loaded;
            }
            __syncwarp();
#pragma unroll 1
            for (int u = u0; u < u1; ++u) {
                const uint32_t slot = loaded % RING;
                if (loaded >= RING) ok = mbar_wait(&bar_q_free[slot], (loaded / RING - 1) & 1, abort_flag) && ok;
                if (ok) {
                    if (lane == 0) {
                        mbar_expect_tx(&bar_q_full[slot], q_bytes);
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb)
                            tma_load_3d(ring + slot * HALF + kb * TILE_BYTES, &map_q, kb * 64, job.kvh * a.group,
                                        job.z.row + (job.from + u) * pairs_nodes, &bar_q_full[slot]);
                    }
                    ++loaded;
                }
                __syncwarp();
            }
            ++jobs;
            t = job.begin + u1;
            if (t < pc.t1) job.next(a, BK, pairs_nodes);
        }
        ring_arrives(bar_q_full, loaded);
        ring_arrives(bar_k_full, k_loaded);
    } else if (warp == MMA_WARP && elect_one()) {
        bool ok = true;
#pragma unroll 1
        for (int t = pc.t0; t < pc.t1;) {
            const int u0 = t - job.begin, u1 = min(job.units, pc.t1 - job.begin), b = jobs & 1;
            ok = mbar_wait(&bar_k_full[b], (jobs >> 1) & 1, abort_flag) && ok;
#pragma unroll 1
            for (int u = u0; u < u1; ++u) {
                const uint32_t at = units_before + (u - u0);          // the block's tiles of rows go to four score tiles in turn
                const uint32_t slot = at % RING, place = at & 3;
                ok = mbar_wait(&bar_q_full[slot], (at / RING) & 1, abort_flag) && ok;
                if (at >= 4) ok = mbar_wait(&bar_free[place], ((at >> 2) - 1) & 1, abort_flag) && ok;
                tc_fence_after();
                if (ok) {
                    issue_scores<KB>(tmem_base + place * 128, smem_u32(k_s + b * HALF), smem_u32(ring + slot * HALF), IDESC);
                    umma_commit(&bar_s[place]);
                }
            }
            units_before += u1 - u0;
            ++jobs;
            t = job.begin + u1;
            if (t < pc.t1) job.next(a, BK, pairs_nodes);
        }
    } else if (warp < MMA_WARP) {
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        bool ok = true;
        int lse_node[4], lse_at[4];          // of the lane's four pairs of a tile: row, and place behind the tile's first
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int pair = lane * 4 + e;
            lse_node[e] = pair < pairs_tile ? pair / a.group : 0x7fffffff;
            lse_at[e] = pair / a.group * a.Hq + pair % a.group;
        }
#pragma unroll 1
        for (int t = pc.t0; t < pc.t1;) {
            const int u0 = t - job.begin, u1 = min(job.units, pc.t1 - job.begin), n = u1 - u0;
            const LlbSpan z = job.z;
            const int key = job.tile * BK + r;
            unsigned long long sum0 = 0, sum1 = 0;
            // minus the lse of four pairs of a tile, minus infinity where there is none
            auto lse_of = [&](int j) -> float4 {
                const int node0 = (job.from + u0 + j) * pairs_nodes, left = j < n ? z.len - node0 : 0;
                const float* from = a.lse + (size_t)(z.row + node0) * a.Hq + job.kvh * a.group;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = lse_node[e] < left ? -from[lse_at[e]] : -INFINITY;
                return make_float4(v[0], v[1], v[2], v[3]);
            };
            const unsigned long long scale2 = llb_pack2(a.scale_log2e, a.scale_log2e);
            const int first = (int)((x - units_before) & 1);          // the group's first tile of the job
            float4 lse = lse_of(first);
#pragma unroll 1
            for (int j = first; j < n; j += 2) {
                const uint32_t at = units_before + j, place = at & 3;
                float* lse_t = lse_s[warp][place >> 1];
                *reinterpret_cast<float4*>(lse_t + lane * 4) = lse;
                __syncwarp();
                lse = lse_of(j + 2);
                ok = mbar_wait(&bar_s[place], (at >> 2) & 1, abort_flag) && ok;
                tc_fence_after();
                if (r == 0) mbar_arrive(&bar_q_free[at % RING]);
                // pairs below `least` belong to rows before the key
                const int node0 = (job.from + u0 + j) * pairs_nodes;
                const int least = (key - z.pos - node0) * a.group;
                const int upto = min(pairs_tile, (z.len - node0) * a.group);
                const bool interior = job.tile * BK + BK - 1 - z.pos - node0 <= 0 && upto == pairs_tile;
                const uint32_t tmem = tmem_base + place * 128 + lanes;
                float s[2][32];
                tmem_ld32_nowait(tmem, *reinterpret_cast<uint32_t(*)[32]>(&s[0][0]));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_wait_ld32(s[c & 1]);
                    if (c < 3) tmem_ld32_nowait(tmem + 32 * (c + 1), *reinterpret_cast<uint32_t(*)[32]>(&s[(c + 1) & 1][0]));
                    float* v = s[c & 1];
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 e = *reinterpret_cast<const float4*>(lse_t + 32 * c + i);
                        llb_unpack2(llb_fma2(llb_pack2(v[i], v[i + 1]), scale2, llb_pack2(e.x, e.y)), v[i], v[i + 1]);
                        llb_unpack2(llb_fma2(llb_pack2(v[i + 2], v[i + 3]), scale2, llb_pack2(e.z, e.w)), v[i + 2], v[i + 3]);
                    }
                    // (Behind the lse: that of a row which is NaN is nothing to keys that the row does not see.  And a key's infinity times the
                    // zeros of columns without a pair is NaN, so these are left out in every tile: 253.6 -> 255.0 us for four portions of
                    // up to 2,048 rows, 28/4 heads of 128; a scan of each job's keys for such numbers instead took 14 us more than that)
                    if (!interior || 32 * c + 32 > pairs_tile) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 32 * c + i >= least && 32 * c + i < upto ? v[i] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        sum0 = llb_add2(sum0, llb_pack2(fast_exp2(v[i]), fast_exp2(v[i + 1])));
                        sum1 = llb_add2(sum1, llb_pack2(fast_exp2(v[i + 2]), fast_exp2(v[i + 3])));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_free[place]);
            }
            float sum, sum_b;
            llb_unpack2(llb_add2(sum0, sum1), sum, sum_b);
            sum += sum_b;
            if (x == 1) sum_s[r] = sum;
            named_barrier(BAR_PAIR, 256);
            if (x == 0) {
                sum += sum_s[r];
                const int part = job.begin < pc.t0 ? 0 : job.begin + job.units > pc.t1 ? 1 : -1;
                if (part >= 0) {
                    m.part[(size_t)(blockIdx.x * 2 + part) * 128 + r] = sum;
                    if (part == 1 && r == 0) llb_leave_open_mass(a, pc, job, true);
                } else if (ok) {
                    llb_add_mass(a, z, job.s, key, job.kvh, sum);
                }
            }
            named_barrier(BAR_PAIR, 256);
            if (threadIdx.x == 0) mbar_arrive(&bar_k_free[jobs & 1]);          // both groups have had all scores of the job
            units_before += n;
            ++jobs;
            t = job.begin + u1;
            if (t < pc.t1) job.next(a, BK, pairs_nodes);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0 && m.p.error_flag) atomicExch(m.p.error_flag, 5);
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// q [T, Hq, hd] in boxes of the group's heads of `nodes` rows.
int make_map_q(const void* q, int T, int Hq, int hd, int group, int nodes, CUtensorMap* out) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return llb_fail("cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)Hq, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)Hq * hd * 2};
    cuuint32_t box[3] = {64u, (cuuint32_t)group, (cuuint32_t)nodes};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult rc = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return llb_fail("cuTensorMapEncodeTiled failed with code %d", (int)rc);
    return 0;
}

// The softmax groups' registers come out of what the block was launched with: a build that gives a thread fewer is refused.
template <int HD> bool registers_suffice() {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, span_attention_tc_kernel<HD>) == cudaSuccess && at.numRegs * 3 >= 104 + 2 * 200;
}
template <int HD>
int launch_tc(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TcParams& p, int blocks, cudaStream_t stream) {
    static const bool suffice = registers_suffice<HD>();
    LLB_REQUIRE(suffice, "span_attention_tcgen05: the kernel was built with too few registers a thread");
    static LlbSharedMemory room;
    cudaError_t e = room.allow(span_attention_tc_kernel<HD>, Shape<HD>::SMEM);
    if (e == cudaSuccess) e = launch_pdl(span_attention_tc_kernel<HD>, dim3(blocks), dim3(NUM_THREADS), Shape<HD>::SMEM, stream, mq, mk, mv, p);
    if (e != cudaSuccess) return llb_fail("span_attention_tcgen05: launch failed: %s", cudaGetErrorString(e));
    return llb_check_launch("span_attention_tcgen05");
}
template <int HD> int launch_mass_tc(const CUtensorMap& mq, const CUtensorMap& mk, const MassArgs& m, int blocks, cudaStream_t stream) {
    static LlbSharedMemory room;
    cudaError_t e = room.allow(span_mass_tc_kernel<HD>, MassShape<HD>::SMEM);
    if (e == cudaSuccess) e = launch_pdl(span_mass_tc_kernel<HD>, dim3(blocks), dim3(NUM_THREADS), MassShape<HD>::SMEM, stream, mq, mk, m);
    if (e != cudaSuccess) return llb_fail("span_mass_tcgen05: launch failed: %s", cudaGetErrorString(e));
    return llb_check_launch("span_mass_tcgen05");
}

}  // namespace

bool llb_span_tc_takes(const LlbSpanArgs& a, const void* q, const void* k, const void* v, const void* out) {
    return (a.hd == 64 || a.hd == 128) && a.group <= 128 && a.page_size % 8 == 0 && a.page_size <= 128 && 128 % a.page_size == 0 &&
           (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 && a.scale_log2e > 0.0f;
}
int llb_span_tc_pairs(int group) { return 128 / group; }

int llb_span_attention_tc(const LlbSpanArgs& a, const void* q, const void* k, const void* v, int blocks, int* error_flag, cudaStream_t stream) {
    TcParams p;
    p.a = a; p.v = (const __nv_bfloat16*)v; p.pairs_nodes = llb_span_tc_pairs(a.group); p.error_flag = error_flag;
    CUtensorMap mq, mk, mv;
    int rc;
    if ((rc = make_map_q(q, a.T, a.Hq, a.hd, a.group, p.pairs_nodes, &mq))) return rc;
    if ((rc = make_map_bf16(k, a.num_slots, (long long)a.Hkv * a.hd, a.page_size, &mk))) return rc;
    if ((rc = make_map_bf16(v, a.num_slots, (long long)a.Hkv * a.hd, a.page_size, &mv))) return rc;
    return a.hd == 64 ? launch_tc<64>(mq, mk, mv, p, blocks, stream) : launch_tc<128>(mq, mk, mv, p, blocks, stream);
}

int llb_span_mass_tc(const LlbSpanArgs& a, const void* q, const void* k, float* part, int blocks, int* error_flag, cudaStream_t stream) {
    MassArgs m;
    m.p.a = a; m.p.v = nullptr; m.p.pairs_nodes = llb_span_tc_pairs(a.group); m.p.error_flag = error_flag;
    m.part = part;
    CUtensorMap mq, mk;
    int rc;
    if ((rc = make_map_q(q, a.T, a.Hq, a.hd, a.group, m.p.pairs_nodes, &mq))) return rc;
    if ((rc = make_map_bf16(k, a.num_slots, (long long)a.Hkv * a.hd, a.page_size, &mk))) return rc;
    return a.hd == 64 ? launch_mass_tc<64>(mq, mk, m, blocks, stream) : launch_mass_tc<128>(mq, mk, m, blocks, stream);
}
