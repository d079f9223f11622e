// Distillation of a retriever's softmax over its candidates from a teacher's top list, forward and backward, for gfx950 (MI355X).
//
//   s_bj = q_b . c_j over T = C + M candidates (the step's C rows, then M constant rows), z = s / temp, l_b = logsumexp_j z_bj
//   t_bi = softmax over the entries i of row b's list of score_bi / teacher_temp   (an index < 0 or a score of -inf is no entry)
//   row_b = sum_i t_bi (log t_bi - z_b,idx(b,i)) + l_b                              (the KL divergence from the teacher's list)
//   loss = mean of row_b over the rows that have an entry; a row without one counts nowhere and receives no gradient
//   g_bj = (softmax(z)_bj - sum_{i: idx(b,i) = j} t_bi) grad_out / rows;  dq = g/temp c, dc = (g/temp)^T q, dtemp = -sum g z / temp
//
// Three products (s, dq, dc) over B x T x d are the work.  fp32 embeddings are multiplied at fp32 accuracy on the bf16 matrix cores:
// x = hi + mid + lo, three bf16 values that carry 24 bits (hi cut, the rest rounded), and the six products of the parts down to
// 2^-16 relative (hi hi, hi mid, mid hi, hi lo, lo hi, mid mid) in fp32 accumulators; what is left out is below 2^-22 of a
// product, random in sign.  Six bf16 MFMAs cost 6/16 of the fp32 MFMA's time for the same product.  bf16 embeddings take
// one product for s; their gradients take two (g in hi + mid, 2^-16 relative, below the 2^-9 of the result's own rounding).
#include "common.h"
#include <type_traits>
#include "../../include/abcsearch.h"

int abc_fail_hip(hipError_t e, const char* where);
int abc_fail_invalid(const char* msg);
int abc_fail_ws(size_t need, size_t have);

typedef __attribute__((ext_vector_type(8))) __bf16 v8bf;
typedef __attribute__((ext_vector_type(2))) __bf16 v2bf;
typedef __attribute__((ext_vector_type(2))) float v2f;
typedef __attribute__((ext_vector_type(4))) unsigned int v4u;

#define DISTILL_MAX_K 1024
#define DISTILL_SEG 4096            // columns of a row that one workgroup turns into gradients

// ---- operands -----------------------------------------------------------------------------------------------------------
// One side of a product: `rows` x K values.  K-contiguous (KC): value (r, k) at row r; K-strided (KS): at row k, column r.
// The candidates lie in two pieces: storage rows below n0 in p0, the others in p1.
struct Side {
    const void* p0;
    const void* p1;
    int64_t n0;                      // storage rows in p0
    int64_t ld;                      // elements between storage rows
    int64_t rows;                    // rows of the product on this side
};

template <bool BF16>
__device__ __forceinline__ const char* storage_row(const Side& s, int64_t i) {
    const char* base = i < s.n0 ? (const char*)s.p0 : (const char*)s.p1;
    return base + (i < s.n0 ? i : i - s.n0) * s.ld * (BF16 ? 2 : 4);
}

// two fp32 values into their bf16 parts, packed (first value low)
template <int PLANES>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[PLANES]) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    w[0] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    float ra = a - __uint_as_float(ua & 0xFFFF0000u), rb = b - __uint_as_float(ub & 0xFFFF0000u);
#pragma unroll
    for (int p = 1; p < PLANES; ++p) {
        const v2bf h = __builtin_convertvector(v2f{ra, rb}, v2bf);
        w[p] = __builtin_bit_cast(uint32_t, h);
        if (p + 1 < PLANES) {
            ra -= __uint_as_float(w[p] << 16);
            rb -= __uint_as_float(w[p] & 0xFFFF0000u);
        }
    }
}

// A tile side in LDS: [plane][k block of 32][row][32 k] bf16, 64 bytes a row, its four 16-byte chunks permuted by (row / 2) % 4 so
// that neither the fragments' reads (8 neighbouring rows, one chunk) nor the writes meet in a bank.
template <int R, int NKB>
__device__ __forceinline__ int lds_at(int plane, int row, int chunk) {
    return (((plane * NKB + (chunk >> 2)) * R + row) << 6) + (((chunk & 3) ^ ((row >> 1) & 3)) << 4);
}

// KC: a thread holds chunks of 8 values along k of one row.  K is a multiple of 8.
template <bool BF16, int PLANES, int R, int NKB>
struct LoadKC {
    static constexpr int CH = NKB * 4, N = R * CH / 256;
    const char* at[N];
    v4u w[N][BF16 ? 1 : 2];
    int row0, chunk;
    __device__ __forceinline__ void init(const Side& s, int64_t r0, int tid) {
        chunk = tid % CH;
        row0 = tid / CH;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int64_t r = r0 + row0 + i * (256 / CH);
            at[i] = r < s.rows ? storage_row<BF16>(s, r) : nullptr;
        }
    }
    __device__ __forceinline__ void load(const Side&, int64_t k0, int64_t k1) {
        const int64_t k = k0 + chunk * 8;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (at[i] && k < k1) {
                const v4u* src = (const v4u*)(at[i] + k * (BF16 ? 2 : 4));
                w[i][0] = src[0];
                if constexpr (!BF16) w[i][1] = src[1];
            } else {
                w[i][0] = v4u{0, 0, 0, 0};
                if constexpr (!BF16) w[i][1] = v4u{0, 0, 0, 0};
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = row0 + i * (256 / CH);
            if constexpr (BF16) {
                *(v4u*)(lds + lds_at<R, NKB>(0, row, chunk)) = w[i][0];
            } else {
                uint32_t o[4][PLANES];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    split_pair<PLANES>(__uint_as_float(w[i][j >> 1][(2 * j) & 3]), __uint_as_float(w[i][j >> 1][(2 * j + 1) & 3]), o[j]);
#pragma unroll
                for (int p = 0; p < PLANES; ++p)
                    *(v4u*)(lds + lds_at<R, NKB>(p, row, chunk)) = v4u{o[0][p], o[1][p], o[2][p], o[3][p]};
            }
        }
    }
};

// KS: a thread holds 8 storage rows (k) of two neighbouring columns and turns them round in its registers.  `rows` is a multiple of
// 2 or storage goes on past it.
template <bool BF16, int PLANES, int R, int NKB>
struct LoadKS {
    static constexpr int CG = R / 2, TASKS = CG * NKB * 4, N = TASKS < 256 ? 1 : TASKS / 256;
    typedef typename std::conditional<BF16, uint32_t, v2f>::type pair_t;
    pair_t w[N][8];
    int64_t col;
    int cg, chunk0;
    bool ok;
    __device__ __forceinline__ void init(const Side& s, int64_t r0, int tid) {
        cg = tid % CG;
        chunk0 = tid / CG;
        col = r0 + cg * 2;
        ok = col < s.rows && (TASKS >= 256 || chunk0 < NKB * 4);
    }
    __device__ __forceinline__ void load(const Side& s, int64_t k0, int64_t k1) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t k = k0 + (chunk0 + i * (256 / CG)) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (ok && k + j < k1) w[i][j] = *(const pair_t*)(storage_row<BF16>(s, k + j) + col * (BF16 ? 2 : 4));
                else if constexpr (BF16) w[i][j] = 0;
                else w[i][j] = v2f{0.f, 0.f};
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) {
        if (TASKS < 256 && chunk0 >= NKB * 4) return;            // a narrow tile leaves some threads without a task
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int chunk = chunk0 + i * (256 / CG);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t o[4][PLANES];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (BF16) o[j][0] = __builtin_amdgcn_perm(w[i][2 * j + 1], w[i][2 * j], c ? 0x07060302u : 0x05040100u);
                    else split_pair<PLANES>(w[i][2 * j][c], w[i][2 * j + 1][c], o[j]);
                }
#pragma unroll
                for (int p = 0; p < PLANES; ++p)
                    *(v4u*)(lds + lds_at<R, NKB>(p, cg * 2 + c, chunk)) = v4u{o[0][p], o[1][p], o[2][p], o[3][p]};
            }
        }
    }
};

struct GemmArgs {
    Side a, b;
    int64_t k;
    int splits;
    int64_t kstep;                   // values of k a split takes (a multiple of the stage)
    int nm, nn;                      // tiles
    void* out;                       // splits == 1: out[m * ldo + n]; otherwise fp32 slabs of `slab` values
    int64_t ldo, slab;
    unsigned* clear;                 // set to zero by the first workgroup (the arrival counter of the next launch), or null
};

// out[m][n] = sum_k A(m, k) B(n, k): tiles of TM x TN, four waves as 2 x 2, 16x16x32 bf16 MFMAs over every pair of planes whose
// indices add up to less than KEEP.  An MFMA rounds its accumulator once (to nearest), so the products of the lower parts have an
// accumulator of their own: the sum of the leading ones is rounded K / 32 times, not 6 K / 32.  One LDS stage; the next stage's values
// are on their way in registers while the current one is multiplied, and two workgroups a CU fill each other's waits.
template <class LA, class LB, int PA, int PB, int KEEP, int TM, int TN, int NKB, bool OUT_BF16>
__global__ __launch_bounds__(256, 2) void distill_gemm_kernel(const GemmArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    char* la = smem_raw;
    char* lb = smem_raw + PA * NKB * TM * 64;
    constexpr int WM = TM / 32, WN = TN / 32, TWO = KEEP > 1;   // 16 x 16 blocks a wave holds along m and n
    if (g.clear && blockIdx.x == 0 && threadIdx.x == 0) *g.clear = 0u;
    // an XCD (every eighth id) takes a run of neighbouring tiles, those of one n tile and split next to each other, so that the larger
    // operand's values are fetched once into its L2
    const int per = g.nm * g.splits, chunk = gridDim.x >> 3;
    const int item = (blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
    if (item >= g.nn * per) return;
    const int tn = item / per, inner = item % per;
    const int tm = inner % g.nm, sp = inner / g.nm;
    const int64_t k0 = sp * g.kstep, k1 = min(g.k, k0 + g.kstep);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l15 = lane & 15, h = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    LA A;
    LB B;
    A.init(g.a, (int64_t)tm * TM, threadIdx.x);
    B.init(g.b, (int64_t)tn * TN, threadIdx.x);
    v4f acc[WM][WN], low[TWO ? WM : 1][TWO ? WN : 1];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j) {
            acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
            if constexpr (TWO) low[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        }
    A.load(g.a, k0, k1);
    B.load(g.b, k0, k1);
    for (int64_t k = k0; k < k1; k += NKB * 32) {
        A.store(la);
        B.store(lb);
        __syncthreads();
        if (k + NKB * 32 < k1) {
            A.load(g.a, k + NKB * 32, k1);
            B.load(g.b, k + NKB * 32, k1);
        }
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            v8bf fb[WN][PB];
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int p = 0; p < PB; ++p) fb[j][p] = *(const v8bf*)(lb + lds_at<TN, NKB>(p, (wn * WN + j) * 16 + l15, kb * 4 + h));
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                v8bf fa[PA];
#pragma unroll
                for (int p = 0; p < PA; ++p) fa[p] = *(const v8bf*)(la + lds_at<TM, NKB>(p, (wm * WM + i) * 16 + l15, kb * 4 + h));
#pragma unroll
                for (int pa = 0; pa < PA; ++pa)
#pragma unroll
                    for (int pb = 0; pb < PB; ++pb)
                        if (pa + pb < KEEP)
#pragma unroll
                            for (int j = 0; j < WN; ++j) {
                                v4f& c = pa + pb == 0 ? acc[i][j] : low[TWO ? i : 0][TWO ? j : 0];
                                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[pa], fb[j][pb], c, 0, 0, 0);
                            }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j) {
            const int64_t n = (int64_t)tn * TN + (wn * WN + j) * 16 + l15;
            if constexpr (TWO) acc[i][j] += low[i][j];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t m = (int64_t)tm * TM + (wm * WM + i) * 16 + 4 * h + r;
                if (m < g.a.rows && n < g.b.rows) {
                    if constexpr (OUT_BF16) ((uint16_t*)g.out)[m * g.ldo + n] = (uint16_t)f32_to_bf16_bits(acc[i][j][r]);
                    else ((float*)g.out)[sp * g.slab + m * g.ldo + n] = acc[i][j][r];
                }
            }
        }
}

// ---- the rows: logsumexp, the teacher's list, the loss -------------------------------------------------------------------
struct RowArgs {
    float* s;                        // slabs [splits][B][lds]; slab 0 holds the sum afterwards
    int splits;
    int64_t slab, lds;
    const float* temp;
    const int64_t* idx;
    const float* score;
    float teacher_temp;
    int64_t B, T;
    int k;
    float* lse;                      // [B]
    float* t;                        // [B][k]; 0 = no entry
    float* row;                      // [B] row losses, then [B] agreement, then [B] 1 where the row has an entry
    float* stat;                     // [0]: 1 / rows that have an entry
    unsigned* cnt;
    float* out_loss;
    float* out_agree;
};

__device__ __forceinline__ float block_max(float v, float* red) {
    for (int m = 32; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = fmaxf(v, red[w]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* red) {     // fixed order
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) v += red[w];
    __syncthreads();
    return v;
}

__global__ __launch_bounds__(512) void distill_row_kernel(const RowArgs a) {
    __shared__ float red[8];
    __shared__ int64_t redi[8];
    __shared__ float ts[DISTILL_MAX_K];
    __shared__ unsigned last;
    const int64_t b = blockIdx.x;
    float* s = a.s + b * a.lds;
    const float t = a.temp[0];
    // one pass: running maximum, its first column, and the sum of exp(z - maximum)
    float mx = -INFINITY, se = 0.f;
    int64_t am = 0;
    bool nan = false;
    for (int64_t j = threadIdx.x * 4; j < a.T; j += 2048) {
        v4f x = *(const v4f*)(s + j);
        for (int p = 1; p < a.splits; ++p) x += *(const v4f*)(s + p * a.slab + j);
        if (a.splits > 1) *(v4f*)(s + j) = x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (j + i >= a.T) break;
            const float z = __fdiv_rn(x[i], t);
            if (z > mx) { se *= expf(mx - z); mx = z; am = j + i; }
            if (z > -INFINITY) se += expf(z - mx);
            nan |= z != z;
        }
    }
    const float top = block_max(mx, red);
    int64_t cand = mx == top && top > -INFINITY ? am : INT64_MAX;
    for (int m = 32; m > 0; m >>= 1) {
        const int lo = __shfl_xor((int)(uint32_t)cand, m, 64), hi = __shfl_xor((int)(cand >> 32), m, 64);
        const int64_t o = ((int64_t)hi << 32) | (uint32_t)lo;
        cand = o < cand ? o : cand;
    }
    if ((threadIdx.x & 63) == 0) redi[threadIdx.x >> 6] = cand;
    __syncthreads();
    for (int w = 0; w < 8; ++w) cand = redi[w] < cand ? redi[w] : cand;
    const float sum = block_sum(mx > -INFINITY ? se * expf(mx - top) : 0.f, red);
    float l = top + logf(sum);
    if (block_max(nan ? 1.f : 0.f, red) > 0.f) l = __uint_as_float(0x7FC00000u);
    // the teacher's list: softmax over its entries, the best of them, the row's loss
    const int64_t* idx = a.idx + b * a.k;
    const float* score = a.score + b * a.k;
    float best = -INFINITY;
    float bad = 0.f, some = 0.f, tnan = 0.f;
    for (int i = threadIdx.x; i < a.k; i += 512) {
        const int64_t at = idx[i];
        const float v = score[i];
        const bool on = at >= 0 && !(v == -INFINITY);
        if (on) {
            some = 1.f;
            if (at >= a.T) bad = 1.f;                            // a column that is not there: the row becomes NaN
            if (!(v < INFINITY)) tnan = 1.f;                     // so does a score that is no number to weigh
            best = fmaxf(best, v);
        }
        ts[i] = on ? v : -INFINITY;
    }
    some = block_max(some, red);
    best = block_max(best, red);
    bad = block_max(fmaxf(bad, tnan), red);
    float e = 0.f;
    int64_t first = INT64_MAX;
    for (int i = threadIdx.x; i < a.k; i += 512) {
        const float v = ts[i];
        if (v == -INFINITY) continue;
        e += expf(__fdiv_rn(v - best, a.teacher_temp));
        if (v == best && i < first) first = i;
    }
    e = block_sum(e, red);
    for (int m = 32; m > 0; m >>= 1) {
        const int o = __shfl_xor((int)(first > 0x7FFFFFFF ? 0x7FFFFFFF : first), m, 64);
        first = o < first ? o : first;
    }
    if ((threadIdx.x & 63) == 0) redi[threadIdx.x >> 6] = first;
    __syncthreads();
    for (int w = 0; w < 8; ++w) first = redi[w] < first ? redi[w] : first;
    const float loge = logf(e);
    float part = 0.f;
    for (int i = threadIdx.x; i < a.k; i += 512) {
        const float v = ts[i];
        float p = 0.f;
        if (v != -INFINITY && bad == 0.f) {
            const float x = __fdiv_rn(v - best, a.teacher_temp);
            p = expf(x) / e;
            if (p > 0.f) part += p * ((x - loge) - __fdiv_rn(s[idx[i]], t));
        }
        a.t[b * a.k + i] = p;
    }
    part = block_sum(part, red);
    if (bad > 0.f) l = __uint_as_float(0x7FC00000u);
    if (threadIdx.x == 0) {
        a.lse[b] = l;
        const bool hit = some > 0.f && bad == 0.f && cand == idx[first];
        __hip_atomic_store(a.row + b, some > 0.f ? part + l : 0.f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.row + a.B + b, hit ? 1.f : 0.f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.row + 2 * a.B + b, some, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the three stores have left (device scope) before the arrival counts
        last = __hip_atomic_fetch_add(a.cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)a.B - 1 ? 1u : 0u;
    }
    __syncthreads();
    if (!last) return;
    // the last row to arrive sums them, in fixed order; its loads go past the caches like the stores did
    float ls = 0.f, hs = 0.f, ns = 0.f;
    for (int64_t i = threadIdx.x; i < a.B; i += 512) {
        ls += __hip_atomic_load(a.row + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        hs += __hip_atomic_load(a.row + a.B + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        ns += __hip_atomic_load(a.row + 2 * a.B + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    ls = block_sum(ls, red);
    hs = block_sum(hs, red);
    ns = block_sum(ns, red);
    if (threadIdx.x == 0) {
        const float n = fmaxf(ns, 1.f);
        a.out_loss[0] = __fdiv_rn(ls, n);
        a.out_agree[0] = __fdiv_rn(hs, n);
        a.stat[0] = __fdiv_rn(1.f, n);
    }
}

// ---- the gradient of the logits ------------------------------------------------------------------------------------------
struct GradArgs {
    const float* s;                  // [B][lds]
    int64_t lds;
    const float* lse;
    const float* t;
    const int64_t* idx;
    const float* has;                // [B]: 1 where the row has an entry
    const float* stat;
    const float* temp;
    const float* grad_out;
    int64_t T, ldg;
    int k;
    float* g;                        // [B][ldg]: (g / temp); zeros from T on
    float* dt;                       // [B][segments]: sums of g z
};

__global__ __launch_bounds__(256) void distill_grad_kernel(const GradArgs a) {
    __shared__ __attribute__((aligned(16))) float buf[DISTILL_SEG];
    __shared__ int li[DISTILL_MAX_K];
    __shared__ float lt[DISTILL_MAX_K];
    __shared__ float red[4];
    const int64_t b = blockIdx.y, j0 = (int64_t)blockIdx.x * DISTILL_SEG;
    const float* s = a.s + b * a.lds + j0;
    float* g = a.g + b * a.ldg + j0;
    const int n = (int)min((int64_t)DISTILL_SEG, a.ldg - j0), valid = (int)max((int64_t)0, min((int64_t)DISTILL_SEG, a.T - j0));
    const bool has = a.has[b] > 0.f;
    const float w = has ? a.grad_out[0] * a.stat[0] : 0.f;
    const float temp = a.temp[0], l = a.lse[b];
    if (has)
        for (int i = threadIdx.x; i < a.k; i += 256) {
            const int64_t at = a.idx[b * a.k + i] - j0;
            const float p = a.t[b * a.k + i];
            li[i] = p != 0.f && at >= 0 && at < valid ? (int)at : -1;
            lt[i] = p;
        }
    for (int i = threadIdx.x * 4; i < n; i += 1024) {
        v4f x = *(const v4f*)(s + i), y;                          // ldg columns are there in s too
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = i + c < valid && has ? expf(__fdiv_rn(x[c], temp) - l) : 0.f;
        *(v4f*)(buf + i) = y;
    }
    __syncthreads();
    if (has)
        for (int i = threadIdx.x; i < a.k; i += 256) {
            const int at = li[i];
            if (at < 0) continue;
            float p = 0.f;
            bool mine = true;                                    // the first of the entries that name this column takes them all
            for (int o = 0; o < a.k; ++o)
                if (li[o] == at) { if (o < i) { mine = false; break; } p += lt[o]; }
            if (mine) buf[at] -= p;
        }
    __syncthreads();
    float dt = 0.f;
    for (int i = threadIdx.x * 4; i < n; i += 1024) {
        const v4f x = *(const v4f*)(s + i);
        v4f y = *(const v4f*)(buf + i);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            y[c] = has ? y[c] * w : 0.f;
            if (i + c < valid && has) dt += y[c] * __fdiv_rn(x[c], temp);
            y[c] = __fdiv_rn(y[c], temp);
        }
        *(v4f*)(g + i) = y;
    }
    dt = block_sum(dt, red);
    if (threadIdx.x == 0) a.dt[b * gridDim.x + blockIdx.x] = dt;
}

// ---- sums of the split products' slabs, and of the temperature's gradient ------------------------------------------------
struct SumArgs {
    const float* part[2];
    void* out[2];
    int64_t n[2];                    // values, a multiple of 4 (0: nothing to do)
    int splits[2];
    int blocks0;                     // workgroups of the first
    const float* dt;
    int64_t ndt;
    const float* temp;
    float* d_temp;                   // null: not wanted
};

template <bool BF16>
__global__ __launch_bounds__(256) void distill_sum_kernel(const SumArgs a) {
    __shared__ float red[4];
    if (blockIdx.x == gridDim.x - 1) {                            // the last workgroup: the temperature
        if (!a.d_temp) return;
        float v = 0.f;
        for (int64_t i = threadIdx.x; i < a.ndt; i += 256) v += a.dt[i];
        v = block_sum(v, red);
        if (threadIdx.x == 0) a.d_temp[0] = -__fdiv_rn(v, a.temp[0]);
        return;
    }
    const int which = (int)blockIdx.x >= a.blocks0;
    const int64_t i = ((int64_t)(blockIdx.x - (which ? a.blocks0 : 0)) * 256 + threadIdx.x) * 4;
    if (i >= a.n[which]) return;
    v4f x = *(const v4f*)(a.part[which] + i);
    for (int p = 1; p < a.splits[which]; ++p) x += *(const v4f*)(a.part[which] + p * a.n[which] + i);
    if constexpr (BF16) {
        uint32_t lo = f32_to_bf16_bits(x[0]) | f32_to_bf16_bits(x[1]) << 16, hi = f32_to_bf16_bits(x[2]) | f32_to_bf16_bits(x[3]) << 16;
        *(uint2*)((uint16_t*)a.out[which] + i) = uint2{lo, hi};
    } else *(v4f*)((float*)a.out[which] + i) = x;
}

// ---- plans ---------------------------------------------------------------------------------------------------------------
struct Plan { int tile, splits; int64_t kstep; int nm, nn; };

// Tiles of 128 x 128 where they fill the chip, 64 x 64 otherwise; k is split until there are two workgroups a CU (512), as long as a
// split keeps four stages.
static Plan plan(int64_t m, int64_t n, int64_t k, int stage) {
    Plan p;
    auto tiles = [&](int t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
    p.tile = m > 64 && n > 64 && tiles(128) * (k / (4 * stage) + 1) >= 512 ? 128 : 64;
    p.nm = (int)((m + p.tile - 1) / p.tile);
    p.nn = (int)((n + p.tile - 1) / p.tile);
    const int64_t stages = (k + stage - 1) / stage;
    int64_t sp = 512 / ((int64_t)p.nm * p.nn);
    if (sp > stages / 4) sp = stages / 4;
    if (sp > 32) sp = 32;
    if (sp < 1) sp = 1;
    const int64_t per = (stages + sp - 1) / sp;
    p.kstep = per * stage;
    p.splits = (int)((stages + per - 1) / per);
    return p;
}

static inline size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

struct FwdLayout { Plan s; int64_t lds; size_t off_lse, off_t, off_row, off_stat, off_cnt, total; };
static int stage_of(int dtype, bool fwd) { (void)fwd; return dtype == ABC_DT_BF16 ? 64 : 32; }

static FwdLayout fwd_layout(int dtype, int64_t B, int64_t T, int d, int k) {
    FwdLayout L;
    L.s = plan(B, T, d, stage_of(dtype, true));
    L.lds = (T + 7) / 8 * 8;
    size_t o = up((size_t)L.s.splits * B * L.lds * 4);
    L.off_lse = o; o += up((size_t)B * 4);
    L.off_t = o; o += up((size_t)B * k * 4);
    L.off_row = o; o += up((size_t)B * 12);
    L.off_stat = o; o += 256;
    L.off_cnt = o; o += 256;
    L.total = o;
    return L;
}

struct BwdLayout { Plan q, p; int64_t ldg; int segs; size_t off_g, off_dt, off_pq, off_pp, total; };
static BwdLayout bwd_layout(int dtype, int64_t B, int64_t C, int64_t T, int d, bool dq, bool dp) {
    BwdLayout L;
    L.ldg = (T + 7) / 8 * 8;
    L.segs = (int)((T + DISTILL_SEG - 1) / DISTILL_SEG);
    L.q = plan(B, d, L.ldg, 32);
    L.p = plan(C, d, B, 32);
    (void)dtype;
    size_t o = up((size_t)B * L.ldg * 4);
    L.off_g = 0;
    L.off_dt = o; o += up((size_t)B * L.segs * 4);
    L.off_pq = o; o += dq && L.q.splits > 1 ? up((size_t)L.q.splits * B * d * 4) : 0;
    L.off_pp = o; o += dp && L.p.splits > 1 ? up((size_t)L.p.splits * C * d * 4) : 0;
    L.total = o;
    return L;
}

static int distill_check(int dtype, int64_t B, int64_t C, int64_t M, int d, int k) {
    if (dtype != ABC_DT_F32 && dtype != ABC_DT_BF16) return abc_fail_invalid("distill: embeddings must be f32 or bf16");
    if (B < 1 || C < 1 || M < 0) return abc_fail_invalid("distill: need at least one query and one candidate");
    if (B > 65535 || C + M > 0x7FFFFFF0ll) return abc_fail_invalid("distill: at most 65535 queries and 2^31 - 16 candidates");
    if (d < 8 || d % 8 || d > 65536) return abc_fail_invalid("distill: d must be a multiple of 8 in [8, 65536]");
    if (k < 1 || k > DISTILL_MAX_K) return abc_fail_invalid("distill: a list has 1 to 1024 entries");
    return ABC_OK;
}

extern "C" size_t abc_distill_workspace_bytes(int dtype, int64_t B, int64_t C, int64_t M, int d, int k) {
    if (distill_check(dtype, B, C, M, d, k)) return 0;
    return fwd_layout(dtype, B, C + M, d, k).total;
}
extern "C" size_t abc_distill_bwd_workspace_bytes(int dtype, int64_t B, int64_t C, int64_t M, int d, int k) {
    if (distill_check(dtype, B, C, M, d, k)) return 0;
    return bwd_layout(dtype, B, C, C + M, d, true, true).total;
}

template <class LA, class LB, int PA, int PB, int KEEP, int T, int NKB, bool OUT_BF16>
static void launch_tile(const GemmArgs& g, hipStream_t st) {
    const unsigned grid = (unsigned)((g.nn * g.nm * g.splits + 7) / 8 * 8);
    hipLaunchKernelGGL((distill_gemm_kernel<LA, LB, PA, PB, KEEP, T, T, NKB, OUT_BF16>), dim3(grid), dim3(256), (PA + PB) * NKB * T * 64, st, g);
}

static GemmArgs gemm_args(const Side& a, const Side& b, int64_t k, const Plan& p, void* out, int64_t ldo, int64_t slab) {
    GemmArgs g;
    g.a = a; g.b = b; g.k = k; g.splits = p.splits; g.kstep = p.kstep; g.nm = p.nm; g.nn = p.nn;
    g.out = out; g.ldo = ldo; g.slab = slab; g.clear = nullptr;
    return g;
}

extern "C" int abc_distill_fwd(int dtype, const void* q, const void* p, const void* memory, const float* temp, const int64_t* teacher_idx,
                               const float* teacher_score, float teacher_temp, int64_t B, int64_t C, int64_t M, int d, int k,
                               float* out_loss, float* out_agree, void* ws, size_t ws_bytes, void* stream) {
    int rc = distill_check(dtype, B, C, M, d, k);
    if (rc) return rc;
    if (!q || !p || (M && !memory) || !temp || !teacher_idx || !teacher_score || !out_loss || !out_agree) return abc_fail_invalid("distill_fwd: null pointer");
    if (((uintptr_t)q | (uintptr_t)p | (uintptr_t)(M ? memory : nullptr)) & 15) return abc_fail_invalid("distill_fwd: embeddings must be 16-byte aligned");
    if (!(teacher_temp > 0.f)) return abc_fail_invalid("distill_fwd: the teacher's temperature must be positive");
    const int64_t T = C + M;
    const FwdLayout L = fwd_layout(dtype, B, T, d, k);
    if (!ws || ws_bytes < L.total) return abc_fail_ws(L.total, ws_bytes);
    if ((uintptr_t)ws & 15) return abc_fail_invalid("distill_fwd: workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    char* w = (char*)ws;
    const Side sq{q, q, B, d, B}, sc{p, memory, C, d, T};
    GemmArgs g = gemm_args(sq, sc, d, L.s, w, L.lds, B * L.lds);
    g.clear = (unsigned*)(w + L.off_cnt);
    if (dtype == ABC_DT_BF16) {
        if (L.s.tile == 128) launch_tile<LoadKC<true, 1, 128, 2>, LoadKC<true, 1, 128, 2>, 1, 1, 1, 128, 2, false>(g, st);
        else launch_tile<LoadKC<true, 1, 64, 2>, LoadKC<true, 1, 64, 2>, 1, 1, 1, 64, 2, false>(g, st);
    } else {
        if (L.s.tile == 128) launch_tile<LoadKC<false, 3, 128, 1>, LoadKC<false, 3, 128, 1>, 3, 3, 3, 128, 1, false>(g, st);
        else launch_tile<LoadKC<false, 3, 64, 1>, LoadKC<false, 3, 64, 1>, 3, 3, 3, 64, 1, false>(g, st);
    }
    RowArgs r;
    r.s = (float*)w; r.splits = L.s.splits; r.slab = B * L.lds; r.lds = L.lds; r.temp = temp; r.idx = teacher_idx; r.score = teacher_score;
    r.teacher_temp = teacher_temp; r.B = B; r.T = T; r.k = k; r.lse = (float*)(w + L.off_lse); r.t = (float*)(w + L.off_t);
    r.row = (float*)(w + L.off_row); r.stat = (float*)(w + L.off_stat); r.cnt = (unsigned*)(w + L.off_cnt);
    r.out_loss = out_loss; r.out_agree = out_agree;
    hipLaunchKernelGGL(distill_row_kernel, dim3((unsigned)B), dim3(512), 0, st, r);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ABC_OK : abc_fail_hip(e, "distill_fwd launch");
}

extern "C" int abc_distill_bwd(int dtype, const void* q, const void* p, const void* memory, const float* temp, const int64_t* teacher_idx,
                               const float* grad_out, int64_t B, int64_t C, int64_t M, int d, int k, void* dq, void* dp, float* d_temp,
                               const void* fwd_ws, size_t fwd_ws_bytes, void* ws, size_t ws_bytes, void* stream) {
    int rc = distill_check(dtype, B, C, M, d, k);
    if (rc) return rc;
    if (!q || !p || (M && !memory) || !temp || !teacher_idx || !grad_out || !fwd_ws) return abc_fail_invalid("distill_bwd: null pointer");
    if (((uintptr_t)q | (uintptr_t)p | (uintptr_t)(M ? memory : nullptr) | (uintptr_t)dq | (uintptr_t)dp) & 15)
        return abc_fail_invalid("distill_bwd: embeddings and gradients must be 16-byte aligned");
    const int64_t T = C + M;
    const FwdLayout F = fwd_layout(dtype, B, T, d, k);
    if (fwd_ws_bytes < F.total) return abc_fail_ws(F.total, fwd_ws_bytes);
    const BwdLayout L = bwd_layout(dtype, B, C, T, d, dq, dp);
    if (!ws || ws_bytes < L.total) return abc_fail_ws(L.total, ws_bytes);
    if (((uintptr_t)ws | (uintptr_t)fwd_ws) & 15) return abc_fail_invalid("distill_bwd: workspaces must be 16-byte aligned");
    if (!dq && !dp && !d_temp) return ABC_OK;
    hipStream_t st = (hipStream_t)stream;
    const char* f = (const char*)fwd_ws;
    char* w = (char*)ws;
    GradArgs a;
    a.s = (const float*)f; a.lds = F.lds; a.lse = (const float*)(f + F.off_lse); a.t = (const float*)(f + F.off_t); a.idx = teacher_idx;
    a.has = (const float*)(f + F.off_row) + 2 * B; a.stat = (const float*)(f + F.off_stat); a.temp = temp; a.grad_out = grad_out;
    a.T = T; a.ldg = L.ldg; a.k = k; a.g = (float*)(w + L.off_g); a.dt = (float*)(w + L.off_dt);
    hipLaunchKernelGGL(distill_grad_kernel, dim3((unsigned)L.segs, (unsigned)B), dim3(256), 0, st, a);
    const bool bf = dtype == ABC_DT_BF16;
    SumArgs sa = {};
    if (dq) {
        const Side ga{a.g, a.g, B, L.ldg, B}, cb{p, memory, C, d, d};
        // the candidates' K-strided side ends at T rows; g's columns from T on are zero and multiply zeros
        GemmArgs g = gemm_args(ga, cb, T, L.q, L.q.splits > 1 ? (void*)(w + L.off_pq) : dq, d, B * d);
        if (!bf) {
            if (L.q.tile == 128) launch_tile<LoadKC<false, 3, 128, 1>, LoadKS<false, 3, 128, 1>, 3, 3, 3, 128, 1, false>(g, st);
            else launch_tile<LoadKC<false, 3, 64, 1>, LoadKS<false, 3, 64, 1>, 3, 3, 3, 64, 1, false>(g, st);
        } else if (L.q.splits > 1) {
            if (L.q.tile == 128) launch_tile<LoadKC<false, 2, 128, 1>, LoadKS<true, 1, 128, 1>, 2, 1, 2, 128, 1, false>(g, st);
            else launch_tile<LoadKC<false, 2, 64, 1>, LoadKS<true, 1, 64, 1>, 2, 1, 2, 64, 1, false>(g, st);
        } else {
            if (L.q.tile == 128) launch_tile<LoadKC<false, 2, 128, 1>, LoadKS<true, 1, 128, 1>, 2, 1, 2, 128, 1, true>(g, st);
            else launch_tile<LoadKC<false, 2, 64, 1>, LoadKS<true, 1, 64, 1>, 2, 1, 2, 64, 1, true>(g, st);
        }
        if (L.q.splits > 1) { sa.part[0] = (const float*)(w + L.off_pq); sa.out[0] = dq; sa.n[0] = B * d; sa.splits[0] = L.q.splits; }
    }
    if (dp) {
        const Side ga{a.g, a.g, B, L.ldg, C}, qb{q, q, B, d, d};
        GemmArgs g = gemm_args(ga, qb, B, L.p, L.p.splits > 1 ? (void*)(w + L.off_pp) : dp, d, C * d);
        if (!bf) {
            if (L.p.tile == 128) launch_tile<LoadKS<false, 3, 128, 1>, LoadKS<false, 3, 128, 1>, 3, 3, 3, 128, 1, false>(g, st);
            else launch_tile<LoadKS<false, 3, 64, 1>, LoadKS<false, 3, 64, 1>, 3, 3, 3, 64, 1, false>(g, st);
        } else if (L.p.splits > 1) {
            if (L.p.tile == 128) launch_tile<LoadKS<false, 2, 128, 1>, LoadKS<true, 1, 128, 1>, 2, 1, 2, 128, 1, false>(g, st);
            else launch_tile<LoadKS<false, 2, 64, 1>, LoadKS<true, 1, 64, 1>, 2, 1, 2, 64, 1, false>(g, st);
        } else {
            if (L.p.tile == 128) launch_tile<LoadKS<false, 2, 128, 1>, LoadKS<true, 1, 128, 1>, 2, 1, 2, 128, 1, true>(g, st);
            else launch_tile<LoadKS<false, 2, 64, 1>, LoadKS<true, 1, 64, 1>, 2, 1, 2, 64, 1, true>(g, st);
        }
        if (L.p.splits > 1) { sa.part[1] = (const float*)(w + L.off_pp); sa.out[1] = dp; sa.n[1] = C * d; sa.splits[1] = L.p.splits; }
    }
    if (sa.n[0] || sa.n[1] || d_temp) {
        sa.blocks0 = (int)((sa.n[0] + 1023) / 1024);
        const int blocks1 = (int)((sa.n[1] + 1023) / 1024);
        sa.dt = a.dt; sa.ndt = B * L.segs; sa.temp = temp; sa.d_temp = d_temp;
        if (bf) hipLaunchKernelGGL(distill_sum_kernel<true>, dim3(sa.blocks0 + blocks1 + 1), dim3(256), 0, st, sa);
        else hipLaunchKernelGGL(distill_sum_kernel<false>, dim3(sa.blocks0 + blocks1 + 1), dim3(256), 0, st, sa);
    }
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ABC_OK : abc_fail_hip(e, "distill_bwd launch");
}
