// Attention over whole requests on CUDA cores, in 32-bit floats: rows with a tree mask or causal ones (see span_attention.cuh), any
// head size up to 256, group and page size, float or bf16 inputs; the joining of cut jobs for this kernel and the tensor-core one;
// and the sums of the weights that keys receive.
//
//     x_ij = scale * q_i . k_j,   m_i = max_j x_ij,   l_i = sum_j 2^(x_ij - m_i),   out_i = sum_j 2^(x_ij - m_i) v_j / l_i
//
// in one pass over the keys with the running maximum and sum (x in base-2 units).  A block of 256 threads holds RB (row, head) pairs
// and walks 64 keys at a time: the tile's K and V go to shared memory as floats, the scores to shared memory for the softmax (whole
// rows are needed there), O stays in registers.  Every thread has 4 rows of the scores and of O, so that a float4 from shared memory
// feeds 16 products or more.  RB is 64, or 16 where requests bring so few rows that most of 64 would stay empty.
#include "cache_calls.h"
#include "memory_ranges.h"
#include "span_attention.cuh"

#include <math.h>

namespace {

constexpr int THREADS = 256;
constexpr int KT = 64;          // keys a tile
constexpr int SP = KT + 4;      // floats from one row of scores to the next

// One head of a slot's row, from column d0 on, four numbers; zeros beyond the head.
template <typename T> __device__ __forceinline__ float4 load4(const T* p, int d, int hd);
template <> __device__ __forceinline__ float4 load4<float>(const float* p, int d, int hd) {
    if (d + 3 < hd && (((uintptr_t)(p + d)) & 15) == 0) return *reinterpret_cast<const float4*>(p + d);
    return make_float4(d < hd ? p[d] : 0.0f, d + 1 < hd ? p[d + 1] : 0.0f, d + 2 < hd ? p[d + 2] : 0.0f, d + 3 < hd ? p[d + 3] : 0.0f);
}
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p, int d, int hd) {
    if (d + 3 < hd && (((uintptr_t)(p + d)) & 7) == 0) {
        const uint2 w = *reinterpret_cast<const uint2*>(p + d);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xffff0000u));
    }
    return make_float4(d < hd ? __bfloat162float(p[d]) : 0.0f, d + 1 < hd ? __bfloat162float(p[d + 1]) : 0.0f,
                       d + 2 < hd ? __bfloat162float(p[d + 2]) : 0.0f, d + 3 < hd ? __bfloat162float(p[d + 3]) : 0.0f);
}
__device__ __forceinline__ bool odd4(const float4& v) {          // an infinity or NaN among them
    return !(fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY && fabsf(v.w) < INFINITY);
}

struct SimtParams {
    LlbSpanArgs a;
    const void* q;
    const void* k;
    const void* v;
};

template <typename T, int RB, int NI>
__global__ void __launch_bounds__(THREADS) span_attention_kernel(const SimtParams p) {
    constexpr int RG = RB / 4, CT = THREADS / RG;      // groups of four rows; threads that share a group's columns
    constexpr int KPT = KT / CT;                       // keys a thread scores
    constexpr int TPR = THREADS / RB;                  // threads a row in the softmax
    constexpr int DPT = RB == 64 ? 4 * NI : NI;        // dimensions of O a thread holds
    const LlbSpanArgs& a = p.a;
    const int hd = a.hd, hd4 = (hd + 3) & ~3, kp = hd4 + 4;
    extern __shared__ __align__(16) float sm[];
    float* q_s = sm;                                   // [RB][hd4]
    float* k_s = q_s + RB * hd4;                       // [KT][kp]
    float* v_s = k_s + KT * kp;                        // [KT][64 * NI]
    float* s_s = v_s + KT * 64 * NI;                   // [RB][SP]
    __shared__ float m_s[RB], l_s[RB], c_s[RB];
    __shared__ int odd_s;
    __shared__ LlbPiece piece_s;
    const int tid = threadIdx.x, ty = tid / CT, tx = tid % CT;
    llb_after_previous();
    if (tid < 32) {
        const LlbPiece pc = llb_piece(a, KT, blockIdx.x, gridDim.x, 1, tid);
        if (tid == 0) piece_s = pc;
    }
    __syncthreads();
    const LlbPiece pc = piece_s;
    LlbJob job = pc.job;
    if (tid == 0) llb_leave_open(a, pc, job, false);
    for (int t = pc.t0; t < pc.t1;) {
        const int rows = job.count(a) * a.group;
        const int k0 = t - job.begin, k1 = min(job.tiles, pc.t1 - job.begin);
        if (k0 >= job.tiles) {
            t = job.begin + job.tiles + a.extra;
            if (t < pc.t1) job.next(a, KT);
            continue;
        }
        const T* qb = (const T*)p.q + ((size_t)(job.z.row + job.first) * a.Hq + job.kvh * a.group) * hd;
        for (int i = tid; i < RB * (hd4 / 4); i += THREADS) {
            const int r = i / (hd4 / 4), d = (i - r * (hd4 / 4)) * 4;
            const float4 v = r < rows ? load4(qb + ((size_t)(r / a.group) * a.Hq + r % a.group) * hd, d, hd) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(q_s + r * hd4 + d) = v;
        }
        if (tid < RB) {
            m_s[tid] = -INFINITY;
            l_s[tid] = tid < rows ? llb_first_sum(a, job.z, job.first + tid / a.group) : 0.0f;
        }
        float o[4][DPT];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < DPT; ++d) o[i][d] = 0.0f;
        // the first so many keys each of the thread's rows sees (-1: it is none of the job's), and where its mask for the others begins
        const unsigned long long* bits = a.mask;
        int own[4];
        size_t mask_at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty * 4 + i, node = job.first + r / a.group;
            own[i] = r >= rows ? -1 : bits ? job.z.pos : job.z.pos + node + 1;
            mask_at[i] = (size_t)(job.z.row + node) * a.words;
        }
        auto sees = [&](int i, int key) {
            if (key < own[i]) return true;
            return bits && own[i] > -1 && key < job.keys && ((bits[mask_at[i] + ((key - job.z.pos) >> 6)] >> ((key - job.z.pos) & 63)) & 1ull);
        };
        for (int kt = k0; kt < k1; ++kt) {
            const int key0 = kt * KT;
            __syncthreads();                           // the tile before has been read
            if (tid == 0) odd_s = 0;
            for (int i = tid; i < KT * 16 * NI; i += THREADS) {
                const int r = i / (16 * NI), d = (i - r * (16 * NI)) * 4, key = key0 + r;
                float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
                const int slot = key < job.keys && d < hd4 ? llb_span_slot(a, job.s, key) : -1;
                if (slot >= 0) {
                    const size_t off = ((size_t)slot * a.Hkv + job.kvh) * hd;
                    kv = load4((const T*)p.k + off, d, hd);
                    vv = load4((const T*)p.v + off, d, hd);
                }
                if (d < hd4) *reinterpret_cast<float4*>(k_s + r * kp + d) = kv;
                *reinterpret_cast<float4*>(v_s + r * (64 * NI) + d) = vv;
            }
            __syncthreads();
            // scores: four rows by KPT keys (CT apart, so that neighbouring threads read neighbouring rows of K)
            unsigned long long x[4][KPT];          // sums of even and of odd dimensions
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) x[i][j] = 0ull;
            for (int d = 0; d < hd4; d += 4) {
                ulonglong2 qv[4], kv[KPT];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const ulonglong2*>(q_s + (ty * 4 + i) * hd4 + d);
#pragma unroll
                for (int j = 0; j < KPT; ++j) kv[j] = *reinterpret_cast<const ulonglong2*>(k_s + (tx + CT * j) * kp + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < KPT; ++j) x[i][j] = llb_fma2(qv[i].y, kv[j].y, llb_fma2(qv[i].x, kv[j].x, x[i][j]));
            }
            const bool inner = key0 + KT <= job.z.pos;          // every row sees the whole tile
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) {
                    const int key = key0 + tx + CT * j;
                    const bool on = inner ? own[i] > -1 : sees(i, key);
                    float lo, hi;
                    llb_unpack2(x[i][j], lo, hi);
                    s_s[(ty * 4 + i) * SP + tx + CT * j] = on ? (lo + hi) * a.scale_log2e : -INFINITY;
                }
            // values of keys that some rows do not see: what is no finite number there must not reach those rows (0 * inf)
            if (!inner)
                for (int i = tid; i < KT * 16 * NI; i += THREADS) {
                    if (odd4(*reinterpret_cast<const float4*>(v_s + i * 4))) odd_s = 1;
                }
            __syncthreads();
            {
                const int r = tid / TPR, c = tid % TPR;
                float* row = s_s + r * SP;
                float top = -INFINITY;
                for (int j = c; j < KT; j += TPR) top = fmaxf(top, row[j]);
#pragma unroll
                for (int w = TPR / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                if (a.scores && job.z.len == 1 && r < rows && job.begin + kt < a.score_tiles)
                    for (int j = c; j < KT; j += TPR) a.scores[((size_t)(job.begin + kt) * a.group + r) * KT + j] = row[j];
                const float m_old = m_s[r], m_new = fmaxf(m_old, top), use = m_new == -INFINITY ? 0.0f : m_new;
                float sum = 0.0f;
                for (int j = c; j < KT; j += TPR) {
                    const float e = exp2f(row[j] - use);
                    row[j] = e;
                    sum += e;
                }
#pragma unroll
                for (int w = TPR / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                __syncwarp();
                if (c == 0) {
                    const float corr = m_old == -INFINITY ? 1.0f : exp2f(m_old - use);          // (nothing so far, or llb_first_sum)
                    c_s[r] = corr;
                    l_s[r] = l_s[r] * corr + sum;
                    m_s[r] = m_new;
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float corr = c_s[ty * 4 + i];
#pragma unroll
                for (int d = 0; d < DPT; ++d) o[i][d] *= corr;
            }
            const bool odd = odd_s != 0;
#pragma unroll 2
            for (int j = 0; j < KT; j += 4) {
                float pr[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(pr[i]) = *reinterpret_cast<const float4*>(s_s + (ty * 4 + i) * SP + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float vv[DPT];
                    if (RB == 64) {
#pragma unroll
                        for (int n = 0; n < NI; ++n)
                            *reinterpret_cast<float4*>(vv + 4 * n) = *reinterpret_cast<const float4*>(v_s + (j + e) * (64 * NI) + n * 64 + tx * 4);
                    } else {
#pragma unroll
                        for (int n = 0; n < NI; ++n) vv[n] = v_s[(j + e) * (64 * NI) + n * 64 + tx];
                    }
                    if (odd) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (!sees(i, key0 + j + e)) continue;          // (a weight of a key that the row sees may be 0 as well)
#pragma unroll
                            for (int d = 0; d < DPT; ++d) o[i][d] = fmaf(pr[i][e], vv[d], o[i][d]);
                        }
                    } else if (DPT % 2 == 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const unsigned long long pp = llb_pack2(pr[i][e], pr[i][e]);
#pragma unroll
                            for (int d = 0; d + 1 < DPT; d += 2)
                                llb_unpack2(llb_fma2(pp, llb_pack2(vv[d], vv[d + 1]), llb_pack2(o[i][d], o[i][d + 1])), o[i][d], o[i][d + 1]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int d = 0; d < DPT; ++d) o[i][d] = fmaf(pr[i][e], vv[d], o[i][d]);
                    }
                }
            }
        }
        const int part = llb_part_of(pc, job);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty * 4 + i;
            if (r >= rows) continue;
            const float l = l_s[r], m = m_s[r];
            const int node = job.first + r / a.group, row = job.z.row + node, head = job.kvh * a.group + r % a.group;
            float* po = a.part_o + (size_t)(blockIdx.x * 2 + max(part, 0)) * (hd4 / 4) * a.rows * 4;
            const float inv = 1.0f / l;
            T* dst = (T*)a.out + ((size_t)row * a.Hq + head) * hd;
            if (RB == 64 && hd % 4 == 0 && (sizeof(T) == 4 ? ((uintptr_t)a.out & 15) == 0 : ((uintptr_t)a.out & 7) == 0)) {
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const int dim = n * 64 + tx * 4;
                    if (dim >= hd) continue;
                    const float* v = o[i] + (RB == 64 ? 4 * n : 0);
                    if (part >= 0) *reinterpret_cast<float4*>(po + ((size_t)(dim >> 2) * a.rows + r) * 4) = make_float4(v[0], v[1], v[2], v[3]);
                    else if (sizeof(T) == 4) *reinterpret_cast<float4*>(dst + dim) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                    else {
                        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0] * inv, v[1] * inv), hi = __floats2bfloat162_rn(v[2] * inv, v[3] * inv);
                        *reinterpret_cast<uint2*>(dst + dim) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
                    }
                }
            } else {
#pragma unroll
                for (int d = 0; d < DPT; ++d) {
                    const int dim = RB == 64 ? (d >> 2) * 64 + tx * 4 + (d & 3) : d * 64 + tx;
                    if (dim >= hd) continue;
                    if (part >= 0) po[((size_t)(dim >> 2) * a.rows + r) * 4 + (dim & 3)] = o[i][d];
                    else dst[dim] = llb_from_float<T>(o[i][d] * inv);
                }
            }
            if (tx == 0) {
                if (part >= 0) {
                    float* ml = a.part_ml + ((size_t)(blockIdx.x * 2 + part) * a.rows + r) * 2;
                    ml[0] = m;
                    ml[1] = l;
                } else if (a.lse) {
                    a.lse[(size_t)row * a.Hq + head] = llb_lse(m, l);
                }
            }
        }
        if (tid == 0 && part == 1) llb_leave_open(a, pc, job, true);
        __syncthreads();                               // the next job's Q, maxima and sums take the places of this one's
        t = job.begin + job.tiles + a.extra;
        if (t < pc.t1) job.next(a, KT);
    }
}

// out = sum_b 2^(m_b - M) O_b / sum_b 2^(m_b - M) l_b over the blocks that hold parts of a job, in their order, with a running maximum
// so that O is asked for together with m and l: a trip to memory after the one for what there is to join.  A warp has 32 rows and four
// dimensions of them; PB parts of PU groups of four dimensions are on their way at once.
template <typename T, int PB, int PU>
__device__ __forceinline__ void join_rows(const LlbSpanArgs& a, const LlbOpen& job, int block, int y, int ny) {
    const int hd = a.hd, pieces = (hd + 3) / 4, groups = (pieces + PU - 1) / PU;
    const int row_groups = (job.rows + 31) / 32;
    for (int i = y * (THREADS / 32) + (threadIdx.x >> 5); i < row_groups * groups; i += ny * (THREADS / 32)) {
        const int r = i / groups * 32 + (threadIdx.x & 31), piece0 = i % groups * PU;
        if (r >= job.rows) continue;
        float x[PU][4], M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int u = 0; u < PU; ++u) x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.0f;
        for (int b0 = 0; b0 < job.parts; b0 += PB) {
            float4 v[PU][PB];
            float2 ml[PB];
#pragma unroll
            for (int e = 0; e < PB; ++e) {
                const int b = b0 + e;
                ml[e] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int u = 0; u < PU; ++u) v[u][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (b >= job.parts) continue;
                const size_t part = (size_t)(block + b) * 2 + (b == 0 ? 1 : 0);
                ml[e] = reinterpret_cast<const float2*>(a.part_ml)[part * a.rows + r];
#pragma unroll
                for (int u = 0; u < PU; ++u)
                    if (piece0 + u < pieces) v[u][e] = reinterpret_cast<const float4*>(a.part_o)[(part * pieces + piece0 + u) * a.rows + r];
            }
            float top = M;
#pragma unroll
            for (int e = 0; e < PB; ++e) top = fmaxf(top, ml[e].x);
            const float keep = M == -INFINITY ? 1.0f : exp2f(M - top);          // (nothing, or a NaN, which stays)
            L *= keep;
            M = top;
#pragma unroll
            for (int u = 0; u < PU; ++u) {
                x[u][0] *= keep; x[u][1] *= keep; x[u][2] *= keep; x[u][3] *= keep;
            }
#pragma unroll
            for (int e = 0; e < PB; ++e) {
                // (a part without visible keys has m = -infinity, l = 0 or llb_first_sum and O = 0; a NaN of another one stays)
                const float w = ml[e].x == -INFINITY ? 1.0f : exp2f(ml[e].x - top);
                L = fmaf(w, ml[e].y, L);
#pragma unroll
                for (int u = 0; u < PU; ++u) {
                    x[u][0] = fmaf(w, v[u][e].x, x[u][0]);
                    x[u][1] = fmaf(w, v[u][e].y, x[u][1]);
                    x[u][2] = fmaf(w, v[u][e].z, x[u][2]);
                    x[u][3] = fmaf(w, v[u][e].w, x[u][3]);
                }
            }
        }
        const int node = r / a.group, row = job.row + node, head = job.kvh * a.group + r - node * a.group;
        const float inv = 1.0f / L;
        if (a.lse && piece0 == 0) a.lse[(size_t)row * a.Hq + head] = llb_lse(M, L);
        T* dst = (T*)a.out + ((size_t)row * a.Hq + head) * hd + piece0 * 4;
        unsigned held0 = 0, held1 = 0;          // two groups of four dimensions leave together
#pragma unroll
        for (int u = 0; u < PU; ++u) {
            const int d = (piece0 + u) * 4;
            if (sizeof(T) == 2 && ((uintptr_t)a.out & 15) == 0 && hd % 8 == 0 && d < hd) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(x[u][0] * inv, x[u][1] * inv), hi = __floats2bfloat162_rn(x[u][2] * inv, x[u][3] * inv);
                const unsigned w0 = *reinterpret_cast<const unsigned*>(&lo), w1 = *reinterpret_cast<const unsigned*>(&hi);
                if (PU == 1) {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
                } else if (u & 1) {
                    *reinterpret_cast<uint4*>(dst + 4 * (u - 1)) = make_uint4(held0, held1, w0, w1);
                } else {
                    held0 = w0;
                    held1 = w1;
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < hd) dst[4 * u + e] = llb_from_float<T>(x[u][e] * inv);
        }
    }
}

// What every key of a request of one row received: the sum of 2^(score - lse) over its kv head's query heads.  The row's lse is what the
// attention kernel left, or, for a cut job, what its parts come to; which that is follows from the lengths, so that these blocks need
// not wait for those that join.
template <typename T, int TILE> __device__ __forceinline__ void mass_of_scores(const LlbSpanArgs& a, int grid, int least, int pair, int y, int ny) {
    __shared__ int before_s, total_s;
    __shared__ float lse_s[128];
    const int s = pair / a.Hkv, kvh = pair - s * a.Hkv;
    const LlbSpan z = llb_span(a, s);
    if (z.len != 1) return;
    // the first key's cache row and what it had, on their way before anything is waited for
    int key = y * THREADS + threadIdx.x;
    int slot = key <= z.pos ? llb_span_slot(a, s, key) : -1;
    float had = slot >= 0 && key < z.pos && a.mass_in ? a.mass_in[(size_t)kvh * a.num_slots + slot] : 0.0f;
    if (threadIdx.x < 32) {
        int before = 0, total = 0;
        for (int i = threadIdx.x; i < a.S; i += 32) {
            const int n = llb_span_tiles(a, llb_span(a, i), TILE);
            total += n;
            if (i < s) before += n;
        }
        before = __reduce_add_sync(0xffffffffu, before);
        total = __reduce_add_sync(0xffffffffu, total);
        if (threadIdx.x == 0) {
            before_s = before;
            total_s = total;
        }
    }
    __syncthreads();
    const int tiles = (z.pos + TILE) / TILE, begin = before_s + kvh * (tiles + a.extra);
    LlbPiece pc;
    pc.total = total_s;
    pc.blocks = min(grid, (pc.total + least - 1) / least);
    const int from = pc.owner(begin), parts = pc.owner(begin + tiles - 1) - from + 1;
    for (int g = threadIdx.x; g < a.group; g += THREADS) {
        float lse;
        if (parts == 1) lse = a.lse[(size_t)z.row * a.Hq + kvh * a.group + g];
        else {
            const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)from * 2 * a.rows + g;
            float M = -INFINITY, L = 0.0f;
#pragma unroll 8
            for (int b = 0; b < parts; ++b) M = fmaxf(M, ml[(size_t)(b == 0 ? 1 : 2 * b) * a.rows].x);
#pragma unroll 8
            for (int b = 0; b < parts; ++b) {
                const float2 x = ml[(size_t)(b == 0 ? 1 : 2 * b) * a.rows];
                L = fmaf(x.x == -INFINITY ? 1.0f : exp2f(x.x - M), x.y, L);
            }
            lse = llb_lse(M, L);
        }
        lse_s[g] = lse;
    }
    __syncthreads();
    for (; key <= z.pos; key += ny * THREADS) {
        if (slot >= 0) {
            const int tile = begin + key / TILE;
            float sum = 0.0f;
            if (tile < a.score_tiles) {
#pragma unroll 8
                for (int g = 0; g < a.group; ++g) sum += exp2f(a.scores[((size_t)tile * a.group + g) * TILE + key % TILE] - lse_s[g]);
            } else {
                // the line is longer than the cache's keys make it (pages outside the cache): there was no place for this one's scores
                const T* q = (const T*)a.q + ((size_t)z.row * a.Hq + kvh * a.group) * a.hd;
                const T* k = (const T*)a.k + ((size_t)slot * a.Hkv + kvh) * a.hd;
#pragma unroll 1
                for (int g = 0; g < a.group; ++g, q += a.hd) {
                    float x = 0.0f;
#pragma unroll 1
                    for (int d = 0; d < a.hd; ++d) x = fmaf(llb_to_float(q[d]), llb_to_float(k[d]), x);
                    sum += exp2f(x * a.scale_log2e - lse_s[g]);
                }
            }
            a.mass[(size_t)kvh * a.num_slots + slot] = had + sum;
        }
        const int next = key + ny * THREADS;
        slot = next <= z.pos ? llb_span_slot(a, s, next) : -1;
        had = slot >= 0 && next < z.pos && a.mass_in ? a.mass_in[(size_t)kvh * a.num_slots + slot] : 0.0f;
    }
}

// The first `blocks * ny` blocks join, the others add up weights, `mass_y` of them a request and kv head.
template <typename T, int TILE>
__global__ void __launch_bounds__(THREADS, 4) span_join_kernel(const LlbSpanArgs a, int blocks, int ny, int mass_y, int least) {
    llb_after_previous();
    const int i = blockIdx.x;
    if (i >= blocks * ny) {
        const int pair = (i - blocks * ny) / mass_y;
        mass_of_scores<T, TILE>(a, blocks, least, pair, i - blocks * ny - pair * mass_y, mass_y);
        return;
    }
    const int y = i / blocks, block = i - y * blocks;
    LlbOpen job;
    const int4 open = reinterpret_cast<const int4*>(a.open)[block];
    job.parts = open.x; job.row = open.y; job.rows = open.z; job.kvh = open.w;
    if (job.parts == 0) return;
    if (job.parts <= 2) join_rows<T, 2, 4>(a, job, block, y, ny);
    else join_rows<T, 8, 1>(a, job, block, y, ny);
}

// The same for requests of any number of rows: 64 keys of one request and kv head stay in shared memory, the rows that see any of them
// go by, up to 64 (row, head) pairs at a time, and their scores are made once more.  A thread adds up four pairs by four keys; the threads
// of a key meet at the end in a fixed order.
struct ColumnParams {
    LlbSpanArgs a;
    const void* q;
    const void* k;
    float* part;            // [2 * blocks, KT]
};
template <typename T>
__global__ void __launch_bounds__(THREADS) span_mass_kernel(const ColumnParams p) {
    constexpr int RB = 64;
    const LlbSpanArgs& a = p.a;
    const int hd = a.hd, hd4 = (hd + 3) & ~3, kp = hd4 + 4, nodes = RB / a.group;
    extern __shared__ __align__(16) float sm[];
    float* q_s = sm;                     // [RB][hd4]
    float* k_s = q_s + RB * hd4;         // [KT][kp]
    __shared__ float lse_s[RB];
    __shared__ float sum_s[16][KT];
    __shared__ LlbMassPiece piece_s;
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    llb_after_previous();
    if (tid < 32) {
        const LlbMassPiece pc = llb_mass_piece(a, KT, nodes, blockIdx.x, gridDim.x, tid);
        if (tid == 0) {
            piece_s = pc;
            llb_leave_open_mass(a, pc.line, pc.job, false);
        }
    }
    __syncthreads();
    const LlbPiece pc = piece_s.line;
    LlbMassJob job = piece_s.job;
    for (int t = pc.t0; t < pc.t1;) {
        const int u0 = t - job.begin, u1 = min(job.units, pc.t1 - job.begin);
        const LlbSpan z = job.z;
        const int key0 = job.tile * KT, keys = z.pos + z.len;
        for (int i = tid; i < KT * (hd4 / 4); i += THREADS) {
            const int r = i / (hd4 / 4), d = (i - r * (hd4 / 4)) * 4;
            const int slot = key0 + r < keys ? llb_span_slot(a, job.s, key0 + r) : -1;
            *reinterpret_cast<float4*>(k_s + r * kp + d) =
                slot >= 0 ? load4((const T*)p.k + ((size_t)slot * a.Hkv + job.kvh) * hd, d, hd) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int u = u0; u < u1; ++u) {
            const int node0 = (job.from + u) * nodes, pairs = min(nodes, z.len - node0) * a.group;
            __syncthreads();
            for (int i = tid; i < RB * (hd4 / 4); i += THREADS) {
                const int r = i / (hd4 / 4), d = (i - r * (hd4 / 4)) * 4;
                *reinterpret_cast<float4*>(q_s + r * hd4 + d) =
                    r < pairs ? load4((const T*)p.q + ((size_t)(z.row + node0 + r / a.group) * a.Hq + job.kvh * a.group + r % a.group) * hd, d, hd)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (tid < RB)
                lse_s[tid] = tid < pairs ? a.lse[(size_t)(z.row + node0 + tid / a.group) * a.Hq + job.kvh * a.group + tid % a.group] : INFINITY;
            __syncthreads();
            unsigned long long x[4][4];          // sums of even and of odd dimensions
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = 0ull;
            for (int d = 0; d < hd4; d += 4) {
                ulonglong2 qv[4], kv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const ulonglong2*>(q_s + (ty * 4 + i) * hd4 + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const ulonglong2*>(k_s + (tx + 16 * j) * kp + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = llb_fma2(qv[i].y, kv[j].y, llb_fma2(qv[i].x, kv[j].x, x[i][j]));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int last = ty * 4 + i < pairs ? z.pos + node0 + (ty * 4 + i) / a.group : -1;          // the last key that the row sees
                const float lse = lse_s[ty * 4 + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float lo, hi;
                    llb_unpack2(x[i][j], lo, hi);
                    if (key0 + tx + 16 * j <= last) sum[j] += exp2f((lo + hi) * a.scale_log2e - lse);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sum_s[ty][tx + 16 * j] = sum[j];
        __syncthreads();
        const int part = job.begin < pc.t0 ? 0 : job.begin + job.units > pc.t1 ? 1 : -1;
        if (tid < KT) {
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) total += sum_s[i][tid];
            if (part >= 0) p.part[(size_t)(blockIdx.x * 2 + part) * KT + tid] = total;
            else llb_add_mass(a, z, job.s, key0 + tid, job.kvh, total);
        }
        if (tid == 0 && part == 1) llb_leave_open_mass(a, pc, job, true);
        __syncthreads();
        t = job.begin + u1;
        if (t < pc.t1) job.next(a, KT, nodes);
    }
}

// The sums of keys whose rows several blocks had, in the blocks' order.
template <int TILE> __global__ void __launch_bounds__(TILE) span_mass_join_kernel(const LlbSpanArgs a, const float* part) {
    llb_after_previous();
    const int4 job = reinterpret_cast<const int4*>(a.open)[blockIdx.x];          // blocks, request, tile, kv head
    if (job.x == 0) return;
    float sum = part[(size_t)(blockIdx.x * 2 + 1) * TILE + threadIdx.x];
#pragma unroll 4
    for (int b = 1; b < job.x; ++b) sum += part[(size_t)(blockIdx.x + b) * 2 * TILE + threadIdx.x];
    llb_add_mass(a, llb_span(a, job.y), job.y, job.z * TILE + threadIdx.x, job.w, sum);
}

template <typename T, int TILE>
int launch_join(const LlbSpanArgs& a, int blocks, int least, cudaStream_t stream) {
    // a warp of the first kind has 32 rows of four dimensions at a time: as many as the average job brings
    const int average = (int)max(1ll, min((long long)a.rows, (long long)a.T * a.group / max(1, a.S)));
    // (small jobs are cut into many parts, of which it takes few groups of dimensions at once)
    const int ny = min(16, llb_ceil_div(llb_ceil_div(average, 32) * llb_ceil_div(a.hd, average <= 128 ? 4 : 16), THREADS / 32));
    int mass_y = 0;
    if (a.scores) {
        const long long keys = (long long)a.max_pages * a.page_size;
        mass_y = (int)max(1ll, min((keys + THREADS - 1) / THREADS, (long long)llb_ceil_div(8 * llb_device_sms(), a.S * a.Hkv)));
    }
    llb_launch(span_join_kernel<T, TILE>, dim3(blocks * ny + a.S * a.Hkv * mass_y), dim3(THREADS), 0, stream, a, blocks, ny, mass_y, least);
    return llb_check_launch("span_join");
}

template <typename T, int RB, int NI>
int launch_attention(const SimtParams& p, int blocks, cudaStream_t stream) {
    const int hd4 = (p.a.hd + 3) & ~3;
    const size_t smem = sizeof(float) * ((size_t)RB * hd4 + KT * (hd4 + 4) + KT * 64 * NI + RB * SP);
    static LlbSharedMemory room;
    cudaError_t e = room.allow(span_attention_kernel<T, RB, NI>, smem);
    if (e != cudaSuccess) return llb_fail("span_attention: cannot opt in to %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    llb_launch(span_attention_kernel<T, RB, NI>, dim3(blocks), dim3(THREADS), smem, stream, p);
    return llb_check_launch("span_attention");
}
template <typename T, int RB>
int launch_attention_hd(const SimtParams& p, int blocks, cudaStream_t stream) {
    if (p.a.hd <= 64) return launch_attention<T, RB, 1>(p, blocks, stream);
    if (p.a.hd <= 128) return launch_attention<T, RB, 2>(p, blocks, stream);
    return launch_attention<T, RB, 4>(p, blocks, stream);
}

}  // namespace

int llb_span_join(const LlbSpanArgs& a, int dtype, int blocks, int tile, int least, cudaStream_t stream) {
    if (dtype == LLB_F32) return launch_join<float, KT>(a, blocks, least, stream);
    return tile == KT ? launch_join<__nv_bfloat16, KT>(a, blocks, least, stream) : launch_join<__nv_bfloat16, 128>(a, blocks, least, stream);
}

namespace {

// (row, head) pairs a job of the CUDA-core kernel holds: 16 where requests bring that many or fewer on average.  (float32, 14/2 heads of 64, 5
// requests of 77 to 1,103 keys, us with 16 | 64: a row each 15 | 20, two 15.4 | 20.5, four 18.5 | 21.5, eight 25 | 22, 64 rows 103 | 48;
// 27 requests: two 26 | 31, four 37 | 33.  Four rows, 28 pairs, go to 64: few requests lose 3 us by that, many gain 4.  Where it changes depends on
// how many blocks have work, which the rule does not ask.)
int simt_rows(int T, int S, int group) { return group <= 16 && (long long)T * group <= 16ll * S ? 16 : 64; }
int simt_blocks() { return min(2 * llb_device_sms(), LLB_SPAN_BLOCKS); }
int tc_blocks() { return min(llb_device_sms(), LLB_SPAN_BLOCKS); }

int check(const LlbSpanArgs& a, int dtype) {
    LLB_REQUIRE(dtype == LLB_F32 || dtype == LLB_BF16, "span_attention: unknown dtype %d", dtype);
    LLB_REQUIRE(a.Hq > 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0 && a.group <= 64, "span_attention: bad head counts %d/%d (at most 64 query heads a kv head)", a.Hq, a.Hkv);
    LLB_REQUIRE(a.hd > 0 && a.hd <= 256, "span_attention: head size %d, up to 256 are supported", a.hd);
    LLB_REQUIRE(a.S >= 0 && a.T >= 0 && a.page_size > 0 && a.max_pages >= 0 && a.num_slots > 0 && (long long)a.max_pages * a.page_size <= (1 << 30),
                "span_attention: bad sizes");
    return 0;
}

// Whether the tensor-core kernels take these sizes (they may still pass a call on, see llb_span_tc_takes).  Where they can they do: 2 rows behind
// 60 keys 9.3 us instead of 11.1 on the CUDA cores, 8 behind 2,048 12.4 instead of 20.7, 27 trees of up to 26 rows 33 instead of 270.
bool tc_sizes(int dtype, int hd, int page_size) {
    return dtype == LLB_BF16 && (hd == 64 || hd == 128) && page_size % 8 == 0 && page_size <= 128 && 128 % page_size == 0;
}
// Scratch: the partial results, the partial sums of the weights, lse, scores.  (Requests share no pages, so that all tiles of one-row
// requests hold no more keys than there are slots, and a piece of a tile each; mass_of_scores makes the others' scores once more.)
// keys: what the requests hold together at most, the cache's rows or their tables' places: a pool may be many times what a call can see.
struct Layout {
    long long part_o, part_ml, open, part_mass, lse, scores, score_tiles, floats;
};
Layout layout(int T, int S, int Hq, int group, int hd, long long keys, int rows, int blocks, int tile, int extra, int mass) {
    Layout l;
    l.part_o = 0;
    l.part_ml = l.part_o + 2ll * blocks * rows * ((hd + 3) & ~3);
    l.open = (l.part_ml + 2ll * blocks * rows * 2 + 3) & ~3ll;
    l.part_mass = l.open + 4ll * blocks;
    l.lse = l.part_mass + (mass == 1 ? 2ll * blocks * 128 : 0);
    l.scores = (l.lse + (mass > 0 ? (long long)T * Hq : 0) + 3) & ~3ll;
    l.score_tiles = mass == 2 ? (keys / tile + (long long)S * (1 + extra)) * (Hq / group) : 0;
    l.floats = l.scores + l.score_tiles * group * tile;
    return l;
}

// mass as llb_span_scratch_floats; tc: on the tensor cores.
int attend(LlbSpanArgs& a, const void* q, const void* k, const void* v, int dtype, float* scratch, int mass, bool tc,
           float** part_mass, int* error_flag, cudaStream_t stream) {
    const int rows = tc ? 2 * llb_span_tc_pairs(a.group) * a.group : simt_rows(a.T, a.S, a.group);
    const int blocks = tc ? tc_blocks() : simt_blocks();
    a.extra = tc ? LLB_SPAN_TC_EXTRA : LLB_SPAN_EXTRA;
    const long long places = min((long long)a.num_slots, (long long)a.S * a.max_pages * a.page_size);
    const Layout l = layout(a.T, a.S, a.Hq, a.group, a.hd, places, rows, blocks, tc ? 128 : KT, a.extra, mass);
    a.rows = rows;
    a.nodes = rows / a.group;
    // (an int numbers the tiles, whatever the lengths on the device say)
    const long long most = min(a.T, a.max_len), keys = (long long)a.max_pages * a.page_size, each = tc ? 128 : KT;
    // (the kernel of portions' weights on the tensor cores has half as many rows a tile)
    LLB_REQUIRE(((most + a.nodes - 1) / a.nodes) * a.S * a.Hkv * ((keys + each - 1) / each + a.extra) * (tc && mass == 1 ? 2 : 1) < (1ll << 31),
                "span_attention: %d requests of up to %lld rows over up to %lld keys are more tiles than one call takes", a.S, most, keys);
    a.part_o = scratch + l.part_o;
    a.part_ml = scratch + l.part_ml;
    a.open = (int*)(scratch + l.open);
    a.lse = mass > 0 ? scratch + l.lse : nullptr;
    a.scores = mass == 2 ? scratch + l.scores : nullptr;
    a.score_tiles = (int)min(l.score_tiles, 0x7fffffffll);
    *part_mass = scratch + l.part_mass;
    a.q = q; a.k = k;
    int rc;
    if (tc) {
        rc = llb_span_attention_tc(a, q, k, v, blocks, error_flag, stream);
        return rc ? rc : llb_span_join(a, dtype, blocks, 128, LLB_SPAN_TC_LEAST, stream);
    }
    SimtParams p;
    p.a = a; p.q = q; p.k = k; p.v = v;
    if (dtype == LLB_F32) rc = rows == 16 ? launch_attention_hd<float, 16>(p, blocks, stream) : launch_attention_hd<float, 64>(p, blocks, stream);
    else rc = rows == 16 ? launch_attention_hd<__nv_bfloat16, 16>(p, blocks, stream) : launch_attention_hd<__nv_bfloat16, 64>(p, blocks, stream);
    return rc ? rc : llb_span_join(a, dtype, blocks, KT, 1, stream);
}

LlbSpanArgs span_args(const LlbSpanCall& s, int max_len) {
    LlbSpanArgs a = {};
    a.out = s.out; a.span_row = s.span_row; a.span_len = s.span_len; a.span_pos = s.span_pos; a.table = s.table;
    a.S = s.S; a.T = s.T; a.max_pages = s.max_pages; a.page_size = s.page_size; a.num_slots = s.num_slots; a.Hq = s.Hq; a.Hkv = s.Hkv; a.hd = s.hd;
    a.page_shift = s.page_size > 0 && (s.page_size & (s.page_size - 1)) == 0 ? __builtin_ctz(s.page_size) : -1;
    a.group = s.Hkv > 0 ? s.Hq / s.Hkv : 0; a.scale_log2e = s.scale * 1.4426950408889634f; a.max_len = max_len;
    return a;
}
// Nothing that the call reads lies under what it writes: the result, and the weights (null: a tree).
int check_apart(const char* what, const LlbSpanCall& s, const unsigned long long* mask, int words, const float* mass, const float* mass_in) {
    const long long e = s.dtype == LLB_F32 ? 4 : 2, rows = (long long)s.T * s.Hq * s.hd * e, plane = (long long)s.num_slots * s.Hkv * s.hd * e;
    const long long spans = 4ll * s.S, weights = 4ll * s.num_slots * s.Hkv;
    return llb_refuse_overlap(what, {{"out", s.out, rows}, {"mass", mass, weights}},
                              {{"q", s.q, rows}, {"k_cache", s.k, plane}, {"v_cache", s.v, plane}, {"mask", mask, 8ll * s.T * words},
                               {"mass_in", mass_in == mass ? nullptr : mass_in, weights}, {"span_row", s.span_row, spans},
                               {"span_len", s.span_len, spans}, {"span_pos", s.span_pos, spans}, {"block_table", s.table, spans * s.max_pages}});
}
bool takes_tc(const LlbSpanArgs& a, const LlbSpanCall& s) {
    return tc_sizes(s.dtype, a.hd, a.page_size) && llb_span_tc_takes(a, s.q, s.k, s.v, s.out);
}

}  // namespace

// Floats of scratch that the calls below take; `keys`: the smaller of num_slots and S * max_pages * page_size (or more); `mass` 0: a tree, 1: with
// the keys' weights, 2: the same where max_len is 1.
LLB_EXPORT long long llb_span_scratch_floats(int dtype, int T, int S, int Hq, int Hkv, int hd, int page_size, int keys, int mass) {
    if (Hkv <= 0 || Hq < Hkv || S <= 0) return 1;
    const int group = Hq / Hkv;
    long long n = layout(T, S, Hq, group, hd, keys, simt_rows(T, S, group), simt_blocks(), KT, LLB_SPAN_EXTRA, mass).floats;
    if (tc_sizes(dtype, hd, page_size) && group <= 128) {
        const long long tc = layout(T, S, Hq, group, hd, keys, 2 * llb_span_tc_pairs(group) * group, tc_blocks(), 128, LLB_SPAN_TC_EXTRA, mass).floats;
        n = tc > n ? tc : n;
    }
    return n;
}

// The calls take one C struct: what a caller from Python pays for an argument of its own (0.12 us) is a tenth of a small call's time.
LLB_EXPORT int llb_tree_attention(const LlbTreeAttention* c, cudaStream_t stream) {
    const LlbSpanCall& s = c->span;
    LlbSpanArgs a = span_args(s, c->words > 0 && c->words <= (1 << 20) ? c->words * 64 : 0);
    if (int rc = check(a, s.dtype)) return rc;
    LLB_REQUIRE(a.max_len > 0 && c->mask && s.scratch, "tree_attention: no mask or no scratch");
    if (a.S == 0 || a.T == 0) return 0;
    if (int rc = check_apart("tree_attention", s, c->mask, c->words, nullptr, nullptr)) return rc;
    a.mask = c->mask;
    a.words = c->words;
    float* unused;
    return attend(a, s.q, s.k, s.v, s.dtype, s.scratch, 0, takes_tc(a, s), &unused, s.error_flag, stream);
}

LLB_EXPORT int llb_paged_attention_mass(const LlbAttentionMass* c, cudaStream_t stream) {
    const LlbSpanCall& s = c->span;
    LlbSpanArgs a = span_args(s, c->max_len);
    if (int rc = check(a, s.dtype)) return rc;
    LLB_REQUIRE(a.max_len > 0 && c->mass && s.scratch, "paged_attention_mass: no weights, no scratch or rows");
    LLB_REQUIRE((long long)a.S * a.Hkv < (1ll << 24), "paged_attention_mass: too many requests");
    if (a.S == 0 || a.T == 0) return 0;
    if (int rc = check_apart("paged_attention_mass", s, nullptr, 0, c->mass, c->mass_in)) return rc;
    const bool single = a.max_len == 1, tc = takes_tc(a, s);
    float* part_mass;
    a.mass_in = c->mass_in;
    a.mass = c->mass;
    if (int rc = attend(a, s.q, s.k, s.v, s.dtype, s.scratch, single ? 2 : 1, tc, &part_mass, s.error_flag, stream)) return rc;
    if (single) return 0;
    if (tc) {
        if (int rc = llb_span_mass_tc(a, s.q, s.k, part_mass, tc_blocks(), s.error_flag, stream)) return rc;
        llb_launch(span_mass_join_kernel<128>, dim3(tc_blocks()), dim3(128), 0, stream, a, (const float*)part_mass);
        return llb_check_launch("span_mass_join");
    }
    ColumnParams p;
    p.a = a; p.q = s.q; p.k = s.k; p.part = part_mass;
    const int hd4 = (a.hd + 3) & ~3;
    const size_t smem = sizeof(float) * ((size_t)64 * hd4 + KT * (hd4 + 4));
    static LlbSharedMemory room_f32, room_bf16;
    auto kernel = s.dtype == LLB_F32 ? span_mass_kernel<float> : span_mass_kernel<__nv_bfloat16>;
    cudaError_t e = (s.dtype == LLB_F32 ? room_f32 : room_bf16).allow(kernel, smem);
    if (e != cudaSuccess) return llb_fail("span_mass: cannot opt in to %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    llb_launch(kernel, dim3(simt_blocks()), dim3(THREADS), smem, stream, p);
    if (int rc = llb_check_launch("span_mass")) return rc;
    llb_launch(span_mass_join_kernel<KT>, dim3(simt_blocks()), dim3(KT), 0, stream, a, (const float*)part_mass);
    return llb_check_launch("span_mass_join");
}
