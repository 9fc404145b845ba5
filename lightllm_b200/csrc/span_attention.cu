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

// Whether row `node` of the request sees key `key` (of those below the request's end).
__device__ __forceinline__ bool sees(const LlbSpanArgs& a, const LlbSpan& z, int node, int key) {
    const int j = key - z.pos;
    if (j < 0) return true;
    if (!a.mask) return j <= node;
    return (a.mask[(size_t)(z.row + node) * a.words + (j >> 6)] >> (j & 63)) & 1ull;
}

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
    if (tid == 0) a.open[blockIdx.x * 4] = -1;
    for (int t = pc.t0; t < pc.t1;) {
        const int rows = job.count(a) * a.group;
        const int k0 = t - job.begin, k1 = min(job.tiles, pc.t1 - job.begin);
        const T* qb = (const T*)p.q + ((size_t)(job.z.row + job.first) * a.Hq + job.kvh * a.group) * hd;
        for (int i = tid; i < RB * (hd4 / 4); i += THREADS) {
            const int r = i / (hd4 / 4), d = (i - r * (hd4 / 4)) * 4;
            const float4 v = r < rows ? load4(qb + ((size_t)(r / a.group) * a.Hq + r % a.group) * hd, d, hd) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(q_s + r * hd4 + d) = v;
        }
        if (tid < RB) {
            m_s[tid] = -INFINITY;
            l_s[tid] = 0.0f;
        }
        float o[4][DPT];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < DPT; ++d) o[i][d] = 0.0f;
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
            float x[4][KPT];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) x[i][j] = 0.0f;
            for (int d = 0; d < hd4; d += 4) {
                float4 qv[4], kv[KPT];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(q_s + (ty * 4 + i) * hd4 + d);
#pragma unroll
                for (int j = 0; j < KPT; ++j) kv[j] = *reinterpret_cast<const float4*>(k_s + (tx + CT * j) * kp + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < KPT; ++j) {
                        x[i][j] = fmaf(qv[i].x, kv[j].x, x[i][j]);
                        x[i][j] = fmaf(qv[i].y, kv[j].y, x[i][j]);
                        x[i][j] = fmaf(qv[i].z, kv[j].z, x[i][j]);
                        x[i][j] = fmaf(qv[i].w, kv[j].w, x[i][j]);
                    }
            }
            const bool inner = key0 + KT <= job.z.pos;          // every row sees the whole tile
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) {
                    const int r = ty * 4 + i, key = key0 + tx + CT * j;
                    const bool on = r < rows && key < job.keys && (inner || sees(a, job.z, job.first + r / a.group, key));
                    s_s[r * SP + tx + CT * j] = on ? x[i][j] * a.scale_log2e : -INFINITY;
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
                if (a.scores && job.z.len == 1 && r < rows)
                    for (int j = c; j < KT; j += TPR) {
                        const int slot = key0 + j < job.keys ? llb_span_slot(a, job.s, key0 + j) : -1;
                        if (slot >= 0) a.scores[(size_t)(job.kvh * a.group + r) * a.num_slots + slot] = row[j];
                    }
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
                    const float corr = m_old == -INFINITY ? 0.0f : exp2f(m_old - use);
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
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int d = 0; d < DPT; ++d) o[i][d] = pr[i][e] == 0.0f ? o[i][d] : fmaf(pr[i][e], vv[d], o[i][d]);
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
            float* po = a.part_o + ((size_t)(blockIdx.x * 2 + max(part, 0)) * a.rows + r) * hd;
            // a row that sees nothing has no sum and gets zeros; one whose visible scores are all minus infinity has none either: NaN
            const float inv = l > 0.0f || m != -INFINITY || job.z.pos > 0 ? 1.0f / l : 0.0f;
            T* dst = (T*)a.out + ((size_t)row * a.Hq + head) * hd;
#pragma unroll
            for (int d = 0; d < DPT; ++d) {
                const int dim = RB == 64 ? (d >> 2) * 64 + tx * 4 + (d & 3) : d * 64 + tx;
                if (dim >= hd) continue;
                if (part >= 0) po[dim] = o[i][d];
                else dst[dim] = llb_from_float<T>(o[i][d] * inv);
            }
            if (tx == 0) {
                if (part >= 0) {
                    float* ml = a.part_ml + ((size_t)(blockIdx.x * 2 + part) * a.rows + r) * 2;
                    ml[0] = m;
                    ml[1] = l;
                } else if (a.lse) {
                    a.lse[(size_t)row * a.Hq + head] = l == 0.0f ? INFINITY : m + log2f(l);
                }
            }
        }
        if (tid == 0 && part == 1) {
            int* d = a.open + blockIdx.x * 4;
            d[0] = job.s; d[1] = job.first; d[2] = job.kvh; d[3] = llb_piece_owner(pc, job.begin + job.tiles - 1);
        }
        t = job.begin + k1;
        if (t < pc.t1) job.next(a, KT);
    }
}

// out = sum_b 2^(m_b - M) O_b / sum_b 2^(m_b - M) l_b over the blocks that hold parts of a job, in their order.  A block takes four
// rows at a time; the parts' factors are worked out once a row.
constexpr int MERGE_ROWS = 4, MERGE_PARTS = 512;
template <typename T>
__global__ void __launch_bounds__(THREADS) span_merge_kernel(const LlbSpanArgs a) {
    __shared__ float w_s[MERGE_ROWS][MERGE_PARTS];
    __shared__ float inv_s[MERGE_ROWS];
    llb_after_previous();
    const int* open = a.open + blockIdx.x * 4;
    const int s = open[0];
    if (s < 0) return;
    const int first = open[1], kvh = open[2], count = open[3] - blockIdx.x + 1;
    const LlbSpan z = llb_span(a, s);
    const int rows = min(a.nodes, z.len - first) * a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto part = [&](int b) { return (size_t)(blockIdx.x + b) * 2 + (b == 0 ? 1 : 0); };
    for (int r0 = blockIdx.y * MERGE_ROWS; r0 < rows; r0 += gridDim.y * MERGE_ROWS) {
        __syncthreads();
        if (warp < MERGE_ROWS && r0 + warp < rows) {
            const int r = r0 + warp;
            float M = -INFINITY;
            for (int b = lane; b < count; b += 32) M = fmaxf(M, a.part_ml[(part(b) * a.rows + r) * 2]);
            M = llb_warp_max(M);
            float L = 0.0f;
            for (int b = lane; b < count; b += 32) {
                const float m = a.part_ml[(part(b) * a.rows + r) * 2], l = a.part_ml[(part(b) * a.rows + r) * 2 + 1];
                const float w = m == -INFINITY ? 0.0f : exp2f(m - M);
                w_s[warp][b] = w;
                // (0 * l: a part without visible keys has l = 0; a NaN of another part stays)
                L += w * l;
            }
            L = llb_warp_sum(L);
            if (lane == 0) {
                inv_s[warp] = L > 0.0f || M != -INFINITY || z.pos > 0 ? 1.0f / L : 0.0f;
                if (a.lse) a.lse[(size_t)(z.row + first + r / a.group) * a.Hq + kvh * a.group + r % a.group] = L == 0.0f ? INFINITY : M + log2f(L);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < MERGE_ROWS * a.hd; i += THREADS) {
            const int w = i / a.hd, d = i - w * a.hd, r = r0 + w;
            if (r >= rows) break;
            float acc = 0.0f;
            for (int b = 0; b < count; ++b) acc = fmaf(w_s[w][b], a.part_o[(part(b) * a.rows + r) * a.hd + d], acc);
            T* dst = (T*)a.out + ((size_t)(z.row + first + r / a.group) * a.Hq + kvh * a.group + r % a.group) * a.hd;
            dst[d] = llb_from_float<T>(acc * inv_s[w]);
        }
    }
}

// What every key of requests of one row received: the sum of 2^(score - lse) over its kv head's query heads.
struct MassParams {
    LlbSpanArgs a;
    const float* mass_in;       // [Hkv, num_slots] or null: zeros
    float* mass;                // [Hkv, num_slots]; may be mass_in
};
__global__ void __launch_bounds__(THREADS) span_mass_of_scores_kernel(const MassParams p) {
    const LlbSpanArgs& a = p.a;
    llb_after_previous();
    const int s = blockIdx.x / a.Hkv, kvh = blockIdx.x - s * a.Hkv;
    const LlbSpan z = llb_span(a, s);
    if (z.len != 1) return;
    const float* lse = a.lse + (size_t)z.row * a.Hq + kvh * a.group;
    for (int key = blockIdx.y * THREADS + threadIdx.x; key <= z.pos; key += gridDim.y * THREADS) {
        const int slot = llb_span_slot(a, s, key);
        if (slot < 0) continue;
        float sum = 0.0f;
        for (int g = 0; g < a.group; ++g) sum += exp2f(a.scores[(size_t)(kvh * a.group + g) * a.num_slots + slot] - lse[g]);
        const size_t at = (size_t)kvh * a.num_slots + slot;
        p.mass[at] = key < z.pos && p.mass_in ? p.mass_in[at] + sum : sum;
    }
}

// The same for requests of any number of rows: 64 keys of one request and kv head stay in shared memory, all rows that see any of them
// go by, 64 (row, head) pairs at a time, and their scores are made once more.  A thread adds up four pairs by four keys; the threads of
// a key meet at the end in a fixed order.
struct ColumnParams {
    LlbSpanArgs a;
    const void* q;
    const void* k;
    const float* mass_in;
    float* mass;
    int blocks_x;
};
template <typename T>
__global__ void __launch_bounds__(THREADS) span_mass_kernel(const ColumnParams p) {
    constexpr int RB = 64;
    const LlbSpanArgs& a = p.a;
    const int hd = a.hd, hd4 = (hd + 3) & ~3, kp = hd4 + 4;
    extern __shared__ __align__(16) float sm[];
    float* q_s = sm;                     // [RB][hd4]
    float* k_s = q_s + RB * hd4;         // [KT][kp]
    __shared__ float lse_s[RB];
    __shared__ float sum_s[16][KT];
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    llb_after_previous();
    // tiles of keys, one request after the other, dealt in turn
    int tile = blockIdx.x;
    for (int s = 0; s < a.S; ++s) {
        const LlbSpan z = llb_span(a, s);
        if (z.len == 0) continue;
        const int keys = z.pos + z.len, tiles = (keys + KT - 1) / KT * a.Hkv;
        for (; tile < tiles; tile += gridDim.x) {
            const int kvh = tile % a.Hkv, key0 = tile / a.Hkv * KT;
            __syncthreads();
            for (int i = tid; i < KT * (hd4 / 4); i += THREADS) {
                const int r = i / (hd4 / 4), d = (i - r * (hd4 / 4)) * 4;
                const int slot = key0 + r < keys ? llb_span_slot(a, s, key0 + r) : -1;
                *reinterpret_cast<float4*>(k_s + r * kp + d) =
                    slot >= 0 ? load4((const T*)p.k + ((size_t)slot * a.Hkv + kvh) * hd, d, hd) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int from = max(0, key0 - z.pos) * a.group, pairs = z.len * a.group;          // rows before see none of the tile
            for (int r0 = from; r0 < pairs; r0 += RB) {
                __syncthreads();
                for (int i = tid; i < RB * (hd4 / 4); i += THREADS) {
                    const int w = i / (hd4 / 4), d = (i - w * (hd4 / 4)) * 4, r = r0 + w;
                    *reinterpret_cast<float4*>(q_s + w * hd4 + d) =
                        r < pairs ? load4((const T*)p.q + ((size_t)(z.row + r / a.group) * a.Hq + kvh * a.group + r % a.group) * hd, d, hd)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                if (tid < RB) {
                    const int r = r0 + tid;
                    lse_s[tid] = r < pairs ? a.lse[(size_t)(z.row + r / a.group) * a.Hq + kvh * a.group + r % a.group] : INFINITY;
                }
                __syncthreads();
                float x[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = 0.0f;
                for (int d = 0; d < hd4; d += 4) {
                    float4 qv[4], kv[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(q_s + (ty * 4 + i) * hd4 + d);
#pragma unroll
                    for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * kp + d);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[i][j] = fmaf(qv[i].x, kv[j].x, x[i][j]);
                            x[i][j] = fmaf(qv[i].y, kv[j].y, x[i][j]);
                            x[i][j] = fmaf(qv[i].z, kv[j].z, x[i][j]);
                            x[i][j] = fmaf(qv[i].w, kv[j].w, x[i][j]);
                        }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int last = z.pos + (r0 + ty * 4 + i) / a.group;          // the last key that the row sees
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (key0 + tx + 16 * j <= last) sum[j] += exp2f(x[i][j] * a.scale_log2e - lse_s[ty * 4 + i]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) sum_s[ty][tx + 16 * j] = sum[j];
            __syncthreads();
            if (tid < KT && key0 + tid < keys) {
                float total = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) total += sum_s[i][tid];
                const int key = key0 + tid, slot = llb_span_slot(a, s, key);
                if (slot >= 0) {
                    const size_t at = (size_t)kvh * a.num_slots + slot;
                    p.mass[at] = key < z.pos && p.mass_in ? p.mass_in[at] + total : total;
                }
            }
        }
        tile -= tiles;
    }
}

template <typename T, int RB, int NI>
int launch_attention(const SimtParams& p, int blocks, cudaStream_t stream) {
    const int hd4 = (p.a.hd + 3) & ~3;
    const size_t smem = sizeof(float) * ((size_t)RB * hd4 + KT * (hd4 + 4) + KT * 64 * NI + RB * SP);
    // (set every time: the attribute belongs to the current device)
    cudaError_t e = cudaFuncSetAttribute(span_attention_kernel<T, RB, NI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
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

int llb_span_merge(const LlbSpanArgs& a, int dtype, int blocks, cudaStream_t stream) {
    LLB_REQUIRE(blocks <= MERGE_PARTS, "span_merge: %d blocks", blocks);
    const int y = min(llb_ceil_div(a.rows, MERGE_ROWS), 16);
    if (dtype == LLB_F32) llb_launch(span_merge_kernel<float>, dim3(blocks, y), dim3(THREADS), 0, stream, a);
    else llb_launch(span_merge_kernel<__nv_bfloat16>, dim3(blocks, y), dim3(THREADS), 0, stream, a);
    return llb_check_launch("span_merge");
}

namespace {

// (row, head) pairs a job of the CUDA-core kernel holds: 16 where requests bring about that many or fewer on average.
int simt_rows(int T, int S, int group) { return group <= 16 && (long long)T * group <= 16ll * S ? 16 : 64; }
int simt_blocks() { return min(2 * llb_device_sms(), MERGE_PARTS); }

int check(const LlbSpanArgs& a, int dtype) {
    LLB_REQUIRE(dtype == LLB_F32 || dtype == LLB_BF16, "span_attention: unknown dtype %d", dtype);
    LLB_REQUIRE(a.Hq > 0 && a.Hkv > 0 && a.Hq % a.Hkv == 0 && a.group <= 64, "span_attention: bad head counts %d/%d (at most 64 query heads a kv head)", a.Hq, a.Hkv);
    LLB_REQUIRE(a.hd > 0 && a.hd <= 256, "span_attention: head size %d, up to 256 are supported", a.hd);
    LLB_REQUIRE(a.S >= 0 && a.T >= 0 && a.page_size > 0 && a.max_pages >= 0 && a.num_slots > 0 && (long long)a.max_pages * a.page_size <= (1 << 30),
                "span_attention: bad sizes");
    LLB_REQUIRE(((long long)a.T / max(1, 64 / a.group) + a.S) * a.Hkv * (((long long)a.max_pages * a.page_size + KT - 1) / KT) < (1ll << 31),
                "span_attention: %d rows over up to %d keys a request are more tiles than one call takes", a.T, a.max_pages * a.page_size);
    return 0;
}

// Whether the tensor-core kernels take these sizes (they may still pass a call on, see llb_span_tc_takes).
bool tc_sizes(int dtype, int hd, int page_size) {
    return dtype == LLB_BF16 && (hd == 64 || hd == 128) && page_size % 8 == 0 && page_size <= 128 && 128 % page_size == 0;
}
// Scratch: the partial results, the blocks' open jobs, the partial sums of the weights, lse, scores.
struct Layout {
    long long part_o, part_ml, open, part_mass, lse, scores, floats;
};
Layout layout(int T, int Hq, int hd, int num_slots, int rows, int blocks, int mass) {
    Layout l;
    l.part_o = 0;
    l.part_ml = l.part_o + 2ll * blocks * rows * hd;
    l.open = l.part_ml + 2ll * blocks * rows * 2;
    l.part_mass = l.open + 4ll * blocks;
    l.lse = l.part_mass + (mass == 1 ? 2ll * blocks * 128 : 0);
    l.scores = l.lse + (mass > 0 ? (long long)T * Hq : 0);
    l.floats = l.scores + (mass == 2 ? (long long)Hq * num_slots : 0);
    return l;
}

// mass as llb_span_scratch_floats; tc: on the tensor cores.
int attend(LlbSpanArgs& a, const void* q, const void* k, const void* v, int dtype, float* scratch, int mass, bool tc, float** part_mass,
           int* error_flag, cudaStream_t stream) {
    const int rows = tc ? 2 * llb_span_tc_pairs(a.group) * a.group : simt_rows(a.T, a.S, a.group);
    const int blocks = tc ? min(llb_device_sms(), MERGE_PARTS) : simt_blocks();
    const Layout l = layout(a.T, a.Hq, a.hd, a.num_slots, rows, blocks, mass);
    a.rows = rows;
    a.nodes = rows / a.group;
    a.part_o = scratch + l.part_o;
    a.part_ml = scratch + l.part_ml;
    a.open = (int*)(scratch + l.open);
    a.lse = mass > 0 ? scratch + l.lse : nullptr;
    a.scores = mass == 2 ? scratch + l.scores : nullptr;
    *part_mass = scratch + l.part_mass;
    int rc;
    if (tc) {
        rc = llb_span_attention_tc(a, q, k, v, blocks, error_flag, stream);
    } else {
        SimtParams p;
        p.a = a; p.q = q; p.k = k; p.v = v;
        if (dtype == LLB_F32) rc = rows == 16 ? launch_attention_hd<float, 16>(p, blocks, stream) : launch_attention_hd<float, 64>(p, blocks, stream);
        else rc = rows == 16 ? launch_attention_hd<__nv_bfloat16, 16>(p, blocks, stream) : launch_attention_hd<__nv_bfloat16, 64>(p, blocks, stream);
    }
    if (rc) return rc;
    return llb_span_merge(a, dtype, blocks, stream);
}

LlbSpanArgs span_args(const void* out, const int* span_row, const int* span_len, const int* span_pos, const int* table, int S, int T,
                      int max_pages, int page_size, int num_slots, int Hq, int Hkv, int hd, float scale, int max_len) {
    LlbSpanArgs a = {};
    a.out = const_cast<void*>(out); a.span_row = span_row; a.span_len = span_len; a.span_pos = span_pos; a.table = table;
    a.S = S; a.T = T; a.max_pages = max_pages; a.page_size = page_size; a.num_slots = num_slots; a.Hq = Hq; a.Hkv = Hkv; a.hd = hd;
    a.group = Hkv > 0 ? Hq / Hkv : 0; a.scale_log2e = scale * 1.4426950408889634f; a.max_len = max_len;
    return a;
}

}  // namespace

// Floats of scratch that the calls below take; `mass` 0: a tree, 1: with the keys' weights, 2: the same where max_len is 1.
LLB_EXPORT long long llb_span_scratch_floats(int dtype, int T, int S, int Hq, int Hkv, int hd, int page_size, int num_slots, int mass) {
    if (Hkv <= 0 || Hq < Hkv || S <= 0) return 1;
    const int group = Hq / Hkv;
    long long n = layout(T, Hq, hd, num_slots, simt_rows(T, S, group), simt_blocks(), mass).floats;
    if (tc_sizes(dtype, hd, page_size) && group <= 128) {
        const long long tc = layout(T, Hq, hd, num_slots, 2 * llb_span_tc_pairs(group) * group, min(llb_device_sms(), MERGE_PARTS), mass).floats;
        n = tc > n ? tc : n;
    }
    return n;
}

// q, out [T, Hq, hd]; caches [num_slots, Hkv, hd]; span arrays [S]; table [S, max_pages]; mask [T, words] 64-bit words.
LLB_EXPORT int llb_tree_attention(const void* q, const void* k, const void* v, void* out, int dtype, const unsigned long long* mask,
                                  int words, const int* span_row, const int* span_len, const int* span_pos, const int* table, int S, int T,
                                  int max_pages, int page_size, int num_slots, int Hq, int Hkv, int hd, float scale, float* scratch,
                                  int* error_flag, cudaStream_t stream) {
    LlbSpanArgs a = span_args(out, span_row, span_len, span_pos, table, S, T, max_pages, page_size, num_slots, Hq, Hkv, hd, scale, 0);
    if (int rc = check(a, dtype)) return rc;
    LLB_REQUIRE(words > 0 && words <= (1 << 20) && mask && scratch, "tree_attention: no mask or no scratch");
    if (S == 0 || T == 0) return 0;
    a.mask = mask;
    a.words = words;
    a.max_len = words * 64;
    float* unused;
    return attend(a, q, k, v, dtype, scratch, 0, tc_sizes(dtype, hd, page_size) && llb_span_tc_takes(a, q, k, v, out), &unused, error_flag, stream);
}

// Causal; mass_in (may be null) and mass [Hkv, num_slots] float, may be the same.
LLB_EXPORT int llb_paged_attention_mass(const void* q, const void* k, const void* v, void* out, int dtype, const float* mass_in, float* mass,
                                        const int* span_row, const int* span_len, const int* span_pos, const int* table, int S, int T,
                                        int max_len, int max_pages, int page_size, int num_slots, int Hq, int Hkv, int hd, float scale,
                                        float* scratch, int* error_flag, cudaStream_t stream) {
    LlbSpanArgs a = span_args(out, span_row, span_len, span_pos, table, S, T, max_pages, page_size, num_slots, Hq, Hkv, hd, scale, max_len);
    if (int rc = check(a, dtype)) return rc;
    LLB_REQUIRE(max_len > 0 && mass && scratch, "paged_attention_mass: no weights, no scratch or rows");
    LLB_REQUIRE((long long)S * Hkv < (1ll << 31), "paged_attention_mass: too many requests");
    if (S == 0 || T == 0) return 0;
    const bool single = max_len == 1;
    const bool tc = tc_sizes(dtype, hd, page_size) && llb_span_tc_takes(a, q, k, v, out);
    float* part_mass;
    if (int rc = attend(a, q, k, v, dtype, scratch, single ? 2 : 1, tc, &part_mass, error_flag, stream)) return rc;
    if (tc && !single) return llb_span_mass_tc(a, q, k, mass_in, mass, part_mass, min(llb_device_sms(), MERGE_PARTS), error_flag, stream);
    const int sms = llb_device_sms();
    if (single) {
        MassParams p;
        p.a = a; p.mass_in = mass_in; p.mass = mass;
        const long long keys = (long long)max_pages * page_size;
        const int y = (int)max(1ll, min((keys + THREADS - 1) / THREADS, (long long)llb_ceil_div(8 * sms, S * Hkv)));
        llb_launch(span_mass_of_scores_kernel, dim3(S * Hkv, y), dim3(THREADS), 0, stream, p);
        return llb_check_launch("span_mass_of_scores");
    }
    ColumnParams p;
    p.a = a; p.q = q; p.k = k; p.mass_in = mass_in; p.mass = mass; p.blocks_x = 2 * sms;
    const int hd4 = (hd + 3) & ~3;
    const size_t smem = sizeof(float) * ((size_t)64 * hd4 + KT * (hd4 + 4));
    auto kernel = dtype == LLB_F32 ? span_mass_kernel<float> : span_mass_kernel<__nv_bfloat16>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return llb_fail("span_mass: cannot opt in to %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    llb_launch(kernel, dim3(p.blocks_x), dim3(THREADS), smem, stream, p);
    return llb_check_launch("span_mass");
}
