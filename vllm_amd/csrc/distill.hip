// Distillation of a retriever's softmax over its candidates from a teacher's top list, forward and backward, for gfx950 (MI355X).
//
//   s_bj = q_b . c_j over T = C + M candidates (the step's C rows, then M constant rows), z = s / temp, l_b = logsumexp_j z_bj
//   t_bi = softmax over the entries i of row b's list of score_bi / teacher_temp   (an index < 0 or a score of -inf is no entry)
//   row_b = sum_i t_bi (log t_bi - z_b,idx(b,i)) + l_b                              (the KL divergence from the teacher's list)
//   loss = mean of row_b over the rows that have an entry; a row without one counts nowhere and receives no gradient
//   g_bj = (softmax(z)_bj - sum_{i: idx(b,i) = j} t_bi) grad_out / rows;  dq = g/temp c, dc = (g/temp)^T q, dtemp = -sum g z / temp
//
// A row's logsumexp stays in two parts, its maximum m and the sum of exp(z - m): in one fp32 number a sum just above 1 would be lost beside a
// large maximum, and with it what a nearly certain row still has to learn (m = 1000: steps of 6e-5).  softmax(z) = exp(z - m) / sum.
//
// A row without an entry has g = 0, and 0 times an infinity or a NaN is not 0: the candidates' product reads such a row's query as zeros
// (a copy that the kernel of g makes beside it, or the split kernel its parts), and its dq is written as zeros.
//
// Three products (s, dq, dc) over B x T x d are the work, on the 16-bit matrix cores (v_mfma_f32_16x16x32):
//
//   fp32, small   x = hi + mid + lo, three bf16 values that carry 24 bits (hi cut, the rest rounded), and the six products of the
//                 parts down to 2^-16 relative (hi hi, hi mid, mid hi, hi lo, lo hi, mid mid): what is left out is below 2^-21 of a
//                 product, random in sign.  Any finite fp32 value (an infinity leaves NaN in the lower parts).
//   fp32, large   x = hi + 2^-11 lo, two fp16 values of 11 bits each (2^-23 of the value), and three products (lo lo, 2^-22, is left
//                 out): half the matrix work for an error of at most 2^-21 of a product, 2^-23 in the root mean square.  Holds for rows whose largest magnitude is in [2^-10, 65000] (a value is carried to 2^-36, 2^-26 of
//                 that, at worst) or zero; unit rows are.  Whether all are is found out while they are read for s; where not, flag is set, and
//                 the same launches once more, which return at once otherwise, take the six products.
//   bf16          one product for s; the gradients take two (g = hi + mid, both rounded: 2^-17 of g at most, below the 2^-8 of the
//                 result's own rounding; with hi cut it would be 2^-16, and twice as many results a place off the nearest).
//
// An MFMA rounds its accumulator once (to nearest), so the products of the lower parts have an accumulator of their own where the result
// is fp32: the sum of the leading ones is rounded K / 32 times, not 6 K / 32.  bf16 gradients have one (2 K / 32 roundings of 2^-24 beside the
// result's own 2^-8) and fit three workgroups a CU (1000 x 5000 x 3584 backward: 185 -> 174 us).
#include "common.h"
#include <type_traits>
#include "../../include/abcsearch.h"

int abc_fail_hip(hipError_t e, const char* where);
int abc_fail_invalid(const char* msg);
int abc_fail_ws(size_t need, size_t have);

typedef __attribute__((ext_vector_type(8))) __bf16 v8bf;
typedef __attribute__((ext_vector_type(2))) __bf16 v2bf;
typedef __attribute__((ext_vector_type(8))) _Float16 v8h;
typedef __attribute__((ext_vector_type(2))) _Float16 v2h;
typedef __attribute__((ext_vector_type(2))) float v2f;
typedef __attribute__((ext_vector_type(4))) unsigned int v4u;
typedef __attribute__((ext_vector_type(2))) unsigned int v2u;

#define DISTILL_MAX_K 1024
#define DISTILL_SEG 2048            // columns of a row that one workgroup of the row and gradient kernels takes
#define G_SCALE 32768.0f            // fp16 gradients are held times 2^15 (softmax - target lies in [-1, 1])
#define H_LOW 65000.0f
#define H_MIN 0x1p-10f

// exp(x) for x <= 0 (and whatever is not a number): 2^n 2^f with n = rint(x log2 e), f to 2^-25
__device__ __forceinline__ float exp_neg(float x) {
    const float n = rintf(x * 1.44269504f);
    const float f = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269502f, -n));      // log2 e in two parts
    return x < -150.f ? 0.f : ldexpf(__builtin_amdgcn_exp2f(f), (int)n);
}

// z of a sum s.  Rounded wherever it is used: fused into a subtraction it would be another number than the one that the row's maximum is.
__device__ __forceinline__ float logit(float s, float inv_temp) {
#pragma clang fp contract(off)
    return s * inv_temp;
}

// ---- operands -----------------------------------------------------------------------------------------------------------
// One side of a product: `rows` x K values.  K-contiguous (KC): value (r, k) at row r; K-strided (KS): at row k, column r.
// The candidates lie in two pieces: storage rows below n0 in p0, the others in p1.
struct Side {
    const void* p0;
    const void* p1;
    int64_t n0;                      // storage rows in p0
    int64_t ld;                      // elements between storage rows
    int64_t rows;                    // rows of the product on this side
    int64_t width;                   // values of a storage row that may be read (a multiple of 8)
};
// Values that lie split into two 16-bit parts: blocks of 32 along the row, 64 bytes of the leading parts and then 64 of the others, so that
// a stage's values of a row are one cache line.  ld counts 16-bit elements (two a value).
__device__ __forceinline__ int64_t split_at(int64_t k) { return (k >> 5) * 128 + (k & 31) * 2; }

template <int ES>
__device__ __forceinline__ const char* storage_row(const Side& s, int64_t i) {
    const char* base = i < s.n0 ? (const char*)s.p0 : (const char*)s.p1;
    return base + (i < s.n0 ? i : i - s.n0) * s.ld * ES;
}

// two fp32 values into their parts, packed (first value low)
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[3]) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    w[0] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    float ra = a - __uint_as_float(ua & 0xFFFF0000u), rb = b - __uint_as_float(ub & 0xFFFF0000u);
    w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{ra, rb}, v2bf));
    ra -= __uint_as_float(w[1] << 16);
    rb -= __uint_as_float(w[1] & 0xFFFF0000u);
    w[2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{ra, rb}, v2bf));
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[2]) {
    const v2h h = __builtin_convertvector(v2f{a, b}, v2h);
    w[0] = __builtin_bit_cast(uint32_t, h);
    const float ra = fmaf((float)h[0], -2048.f, a * 2048.f), rb = fmaf((float)h[1], -2048.f, b * 2048.f);
    w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{ra, rb}, v2h));
}
// two fp32 values as two bf16 parts each, packed, to 2^-17 of the value
__device__ __forceinline__ void split_round(float a, float b, uint32_t (&w)[2]) {
    w[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
    const float ra = a - __uint_as_float(w[0] << 16), rb = b - __uint_as_float(w[0] & 0xFFFF0000u);
    w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{ra, rb}, v2bf));
}

// A converted tile side in LDS: [part][row][32 k], 64 bytes a row, four 16-byte chunks permuted with the row.  A 16-byte access of
// a wave goes in phases of 16 lanes, {0-3, 12-15, 20-27} and {4-11, 16-19, 28-31} and the same of the upper half; a phase of a fragment's
// read holds rows r, r + 12 of one chunk and r + 4, r + 8 of the next, and with -(row / 4) mod 4 those four never share a bank.
template <int R>
__device__ __forceinline__ int lds_at(int part, int row, int chunk) {
    return ((part * R + row) << 6) + (((chunk ^ (0 - (row >> 2))) & 3) << 4);
}

__device__ __forceinline__ uint32_t lds_address(const char* lds) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds; }

// The loaders of fp32 sides hold DEPTH stages of a side's values in registers (load), and put them into LDS, turned and split into PARTS
// as the matrix instructions take them (three bf16 or two fp16 parts), in UNITS steps (store).  Rows past the end are the last row again:
// their results are not kept.  TAIL: the stage may reach past k1, where the values are zero.  NT: the workgroup's threads.

// KC: the lanes of a wave read whole 128-byte lines: 16 bytes of a row each, 8 neighbouring lanes a row's stage.  RANGE: keeps the largest
// magnitude of what it reads.
template <int PARTS, int R, int DEPTH, int NT = 256, bool RANGE = false>
struct LoadKC {
    static constexpr bool KC = true;
    static constexpr int N = R * 8 / NT, UNITS = N, LOADS = N;
    const char* at[N];
    v4u w[DEPTH][N];
    float top[RANGE ? N : 1];
    int row0, sub;
    static __host__ __device__ constexpr int tile_index(int lds_row) { return lds_row; }
    __device__ __forceinline__ void init(const Side& s, int64_t r0, int tid) {
        sub = tid % 8;
        row0 = tid / 8;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t r = r0 + row0 + i * (NT / 8);
            at[i] = storage_row<4>(s, r < s.rows ? r : s.rows - 1) + sub * 16;
            if constexpr (RANGE) top[i] = 0.f;
        }
    }
    template <bool TAIL>
    __device__ __forceinline__ void load(int d, const Side& s, int64_t k0, int64_t k1) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!TAIL || k0 + sub * 4 < k1) w[d][i] = *(const v4u*)(at[i] + k0 * 4);
            else w[d][i] = v4u{0, 0, 0, 0};
        }
    }
    // where the other side is zero from k1 on: the row's last values again, without a branch
    __device__ __forceinline__ void load_held(int d, const Side& s, int64_t k0, int64_t k1) {
        const int k = min((int)k0, (int)k1 - 4 - sub * 4);        // (at[] has the lane's four values in it)
#pragma unroll
        for (int i = 0; i < N; ++i) w[d][i] = *(const v4u*)(at[i] + (int64_t)k * 4);
    }
    __device__ __forceinline__ void store(int d, int i, char* lds) {
        const v4u x = w[d][i];
        uint32_t o[2][PARTS];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float u = __uint_as_float(x[2 * j]), v = __uint_as_float(x[2 * j + 1]);
            split_pair(u, v, o[j]);
            if constexpr (RANGE) top[i] = fmaxf(fmaxf(fabsf(u), fabsf(v)), top[i]);
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) *(v2u*)(lds + lds_at<R>(p, row0 + i * (NT / 8), sub >> 1) + (sub & 1) * 8) = v2u{o[0][p], o[1][p]};
    }
    // the values of a stage, not before here: the compiler would wait for them at the top of the stage
    __device__ __forceinline__ void pin(int d) {
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[d][i]));
    }
    // whether a row that this thread has a part in does not fit the fp16 parts
    __device__ __forceinline__ bool outside() {
        bool bad = false;
        if constexpr (RANGE)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float v = top[i];
#pragma unroll
                for (int m = 1; m < 8; m <<= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
                bad |= v > 0.f && !(v >= H_MIN && v <= H_LOW);
            }
        return bad;
    }
};

// KS: a thread holds 8 storage rows (k) of two neighbouring columns (one, where the tile has too few for the threads) and turns them
// round in its registers.  Columns 2x and 2x + 1 of 32 lie in LDS rows x and 16 + x, so that a wave's writes go to neighbouring rows,
// and a lane's accumulators of two neighbouring blocks are neighbours in memory again.
template <int PARTS, int R, int DEPTH, int NT = 256>
struct LoadKS {
    static constexpr bool KC = false;
    static constexpr int COLS = R * 2 < NT ? 1 : 2, CG = R / COLS, UNITS = COLS, LOADS = 8;
    static_assert(CG * 4 == NT, "a tile that does not fit the threads");
    typedef typename std::conditional<COLS == 2, v2f, float>::type piece_t;
    piece_t w[DEPTH][8];
    int64_t off;
    int row, chunk;
    static __host__ __device__ constexpr int tile_index(int r) { return COLS == 1 ? r : (r & ~31) + ((r & 15) << 1) + ((r >> 4) & 1); }
    __device__ __forceinline__ void init(const Side& s, int64_t r0, int tid) {
        const int cg = tid % CG;
        chunk = __builtin_amdgcn_readfirstlane(tid / CG);         // a wave's storage rows are scalar
        row = COLS == 1 ? cg : (cg >> 4) * 32 + (cg & 15);
        const int64_t last = (s.rows - 1) & ~(int64_t)(COLS - 1), col = r0 + cg * COLS;   // (`rows` is even or storage goes on past it)
        off = (col < last ? col : last) * 4;
    }
    template <bool TAIL>
    __device__ __forceinline__ void load(int d, const Side& s, int64_t k0, int64_t k1) {
        const int64_t k = k0 + chunk * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!TAIL || k + j < k1) w[d][j] = *(const piece_t*)(storage_row<4>(s, k + j) + off);
            else w[d][j] = piece_t{};
        }
    }
    __device__ __forceinline__ void load_held(int d, const Side& s, int64_t k0, int64_t k1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[d][j] = *(const piece_t*)(storage_row<4>(s, min(k0 + chunk * 8 + j, k1 - 1)) + off);
    }
    __device__ __forceinline__ float value(const piece_t& x, int c) const {
        if constexpr (COLS == 2) return x[c];
        else return x;
    }
    __device__ __forceinline__ void store(int d, int c, char* lds) {
        uint32_t o[4][PARTS];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_pair(value(w[d][2 * j], c), value(w[d][2 * j + 1], c), o[j]);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) *(v4u*)(lds + lds_at<R>(p, row + c * 16, chunk)) = v4u{o[0][p], o[1][p], o[2][p], o[3][p]};
    }
    __device__ __forceinline__ void pin(int d) {
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(w[d][j]));
    }
    __device__ __forceinline__ bool outside() { return false; }
};

// ---- sides that need no conversion: straight from memory into LDS -------------------------------------------------------
// 16 bytes a lane, 1 KB a wave's instruction, no register on the way.  A stage is 32 values of k; PARTS of it lie one behind the other.
// All of a workgroup's waves take part.  `tail` brings a last, partial stage through registers, with zeros past k1.
// In asm, for the compiler, where it knows of such a load, gives up counting the others (each wait becomes one for all).  It then counts
// too few on their way, so that its own waits are only longer; for these loads every user waits itself, and before the workgroup ends.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"                    // (m0 is set here and used here alone)
__device__ __forceinline__ void to_lds(const char* src, char* lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds_address(lds)) : "memory", "m0");
}
#pragma clang diagnostic pop

// Rows of a stage are one cache line, 128 bytes: 64 values, or 32 in two parts.  Their eight chunks of 16 bytes are permuted with the
// row (chunk ^ row / 2), which keeps the 16 lanes of a read's phase in different banks; a fragment is one 16-byte read.
template <int PARTS, int R, int NT = 256>
struct DmaKC {
    static constexpr bool KC = true;
    static constexpr int KB = 2 / PARTS, BYTES = R * 128, PASS = NT / 8, N = R / PASS;   // KB: blocks of 32 values a stage; PASS: rows an instruction of all waves
    const char* at[N];
    int chunk, row0, wave;
    __device__ __forceinline__ void init(const Side& s, int64_t r0, int tid) {
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int lane = tid & 63;
        row0 = wave * 8 + (lane >> 3);
        chunk = (lane ^ (row0 >> 1)) & 7;                         // (PASS rows on, the same)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t r = r0 + row0 + i * PASS;
            at[i] = storage_row<2>(s, r < s.rows ? r : s.rows - 1) + chunk * 16;
        }
    }
    __device__ __forceinline__ void issue(const Side&, int64_t k, char* lds) {
#pragma unroll
        for (int i = 0; i < N; ++i) to_lds(at[i] + k * (2 * PARTS), lds + (i * PASS + wave * 8) * 128);
    }
    __device__ __forceinline__ void tail(const Side&, int64_t k, int64_t k1, char* lds) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v4u x = {0, 0, 0, 0};
            if (k + (PARTS == 2 ? chunk & 3 : chunk) * 8 < k1) x = *(const v4u*)(at[i] + k * (2 * PARTS));
            *(v4u*)(lds + (row0 + i * PASS) * 128 + ((chunk ^ (row0 >> 1)) & 7) * 16) = x;
        }
    }
    // the fragments of N blocks of 16 rows from `block` on; which: the part, or the block of 32 values
    template <class F, int J>
    static __device__ __forceinline__ void frags(F (&out)[J], const char* lds, int which, int block, int lane) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int row = (block + j) * 16 + (lane & 15);
            out[j] = *(const F*)(lds + row * 128 + (((which * 4 + (lane >> 4)) ^ (row >> 1)) & 7) * 16);
        }
    }
};

// storage rows (k) lie in LDS as they are, R values each; ds_read_b64_tr_b16 turns 4 of them by 16 columns on the way to a fragment.
// 16-byte chunks are permuted with the row so that the 16 rows of a read spread over all banks.
template <int PARTS, int R, int NT = 256>
struct DmaKS {
    static constexpr bool KC = false;
    static constexpr int KB = 1, CH = R / 8, PER = 64 / CH, PASS = PER * (NT / 64), EACH = 32 / PASS, BYTES = PARTS * R * 64;   // PER: rows an instruction of a wave
    int64_t off;
    int row0, wave;
    static __device__ __forceinline__ int swz(int k) {
        return R >= 128 ? 2 * ((k & 3) | ((k >> 1) & 4)) : 2 * (((k >> 1) & 1) | ((k >> 2) & 2));
    }
    __device__ __forceinline__ void init(const Side& s, int64_t r0, int tid) {
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int lane = tid & 63;
        row0 = wave * PER + lane / CH;                            // and PASS rows on: the permutation repeats every 16 rows
        int64_t col = r0 + ((lane % CH) ^ swz(row0)) * 8;
        if (col > s.width - 8) col = s.width - 8;
        off = PARTS == 2 ? split_at(col) : col * 2;
    }
    __device__ __forceinline__ void issue(const Side& s, int64_t k, char* lds) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const char* src = storage_row<2>(s, k + row0 + e * PASS) + off;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) to_lds(src + p * 64, lds + (p * 32 + wave * PER + e * PASS) * R * 2);
        }
    }
    __device__ __forceinline__ void tail(const Side& s, int64_t k, int64_t k1, char* lds) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int row = row0 + e * PASS;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                v4u x = {0, 0, 0, 0};
                if (k + row < k1) x = *(const v4u*)(storage_row<2>(s, k + row) + off + p * 64);
                *(v4u*)(lds + (p * 32 + row) * R * 2 + (lane % CH) * 16) = x;
            }
        }
    }
    // A block's 16 columns are two chunks; lane (i, c) of it addresses row 8 c + i / 4 and, by offset, the row four on.  (In asm, with its
    // wait inside: for the builtin the compiler waits for every load to LDS that is on its way.)
    template <class F, int N>
    static __device__ __forceinline__ void frags(F (&out)[N], const char* lds, int part, int block, int lane) {
        static_assert(N == 2 || N == 4, "");
        const int i = lane & 15, row = (lane >> 4) * 8 + (i >> 2);
        const uint32_t at = lds_address(lds) + (part * 32 + row) * R * 2 + (i & 1) * 8;
        uint32_t x[N];
        v2u h[2 * N];
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = at + ((((block + j) * 2 + ((i & 3) >> 1)) ^ swz(row)) << 4);
        if constexpr (N == 4)
            asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(h[0]), "=&v"(h[1]), "=&v"(h[2]), "=&v"(h[3]), "=&v"(h[4]), "=&v"(h[5]), "=&v"(h[6]), "=&v"(h[7])
                         : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "n"(8 * R) : "memory");
        else
            asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                         "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(h[0]), "=&v"(h[1]), "=&v"(h[2]), "=&v"(h[3]) : "v"(x[0]), "v"(x[1]), "n"(8 * R) : "memory");
#pragma unroll
        for (int j = 0; j < N; ++j) {
            union { F f; v2u w[2]; } u;
            u.w[0] = h[2 * j];
            u.w[1] = h[2 * j + 1];
            out[j] = u.f;
        }
    }
};

struct GemmArgs {
    Side a, b;
    int64_t k;
    int splits;
    int64_t kstep;                   // values of k a split takes (a multiple of the stage)
    int nm, nn;                      // tiles
    void* out;                       // out[m * ldo + n]; splits > 1: fp32 slabs of `slab` values
    int64_t ldo, slab;
    float scale;                     // of every sum
    const float *f0, *f1, *f2;       // splits == 1, f0 given: times f0[0] f1[0] / f2[0]
    float* seg;                      // splits == 1, given: every wave's part of a row's statistics, [rows][segs][4] (RowArgs), z = value / f2[0]
    int segs;
    const float* live;               // given: a row of A's side where it is not above 0 gives zeros
};

// reductions over the 16 lanes that hold a row of an accumulator; every lane gets the result
template <int CTRL>
__device__ __forceinline__ int dpp16(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, true); }
#define DPP16(x, OP) do { x = OP(x, DPP16_AS(x, 0xB1)); x = OP(x, DPP16_AS(x, 0x4E)); x = OP(x, DPP16_AS(x, 0x141)); x = OP(x, DPP16_AS(x, 0x140)); } while (0)
__device__ __forceinline__ float add_op(float a, float b) { return a + b; }
__device__ __forceinline__ float max16(float x) {
#define DPP16_AS(v, c) __int_as_float(dpp16<c>(__float_as_int(v)))
    DPP16(x, fmaxf);
    return x;
}
__device__ __forceinline__ float sum16(float x) {
    DPP16(x, add_op);
    return x;
#undef DPP16_AS
}
__device__ __forceinline__ int min16(int x) {
#define DPP16_AS(v, c) dpp16<c>(v)
    DPP16(x, min);
    return x;
#undef DPP16_AS
}

__device__ __forceinline__ float factor_of(const float* f0, const float* f1, const float* f2) { return __fdiv_rn(f0[0] * f1[0], f2[0]); }

// out[m][n] = sum_k A(m, k) B(n, k): tiles of TM x TN by NT threads, waves as NT / 128 x 2, 16x16x32 MFMAs over every pair of parts whose
// indices add up to less than KEEP, in stages of 32 or 64 values.  Three ways to bring a stage's values:
//
//   Cfg        both sides fp32, through registers: while a stage is multiplied out of one LDS buffer, the next one's values go from
//              registers into the other, a step of it after each row of MFMAs (the vector unit works in their shadow), and the loads of
//              DEPTH stages further on are on their way: one barrier a stage, which waits for LDS alone.  LBUF 1: one buffer and two
//              barriers, where two would leave a CU one workgroup.
//   CfgMix     A straight into LDS, B as above.
//   CfgDma     both straight into LDS.
//
// FROM: the step (row of MFMAs) of a stage from which on the next stage's values go to LDS.  The later, the longer their loads may
// take, and the less of the conversion lies in the MFMAs' shadow.
template <class LA_, class LB_, int PARTS_, int TILE_, int DEPTH_, int LBUF_, int FROM_>
struct Cfg {
    typedef LA_ LA;
    typedef LB_ LB;
    static constexpr int NT = 256, PA = PARTS_, PB = PARTS_, KEEP = PARTS_, TM = TILE_, TN = TILE_, DEPTH = DEPTH_, LBUF = LBUF_, FROM = FROM_, KIND = 0;
    static constexpr bool F16 = false, OUT_BF16 = false, LOW = true, SCORES = LA::KC && LB::KC;
    static constexpr int LDS = LBUF * (PA * TM + PB * TN) * 64;
};
template <class DA_, class LB_, int TM_, int TN_, int NT_, int FROM_>
struct CfgMix {
    typedef DA_ DA;
    typedef LB_ LB;
    static constexpr int NT = NT_, PA = 2, PB = 2, KEEP = 2, TM = TM_, TN = TN_, FROM = FROM_, KIND = 1;
    static constexpr bool F16 = true, OUT_BF16 = false, LOW = true, SCORES = LB::KC;
    static constexpr int BUF = DA::BYTES + PB * TN * 64, LDS = 2 * BUF;
    static_assert(DA::KC && DA::KB == 1, "");
};
template <class DA_, class DB_, int PA_, int PB_, int TM_, int TN_, int NT_, bool F16_, bool OUT_BF16_>
struct CfgDma {
    typedef DA_ DA;
    typedef DB_ DB;
    static constexpr int NT = NT_, PA = PA_, PB = PB_, KEEP = PA_, TM = TM_, TN = TN_, BUF = DA::BYTES + DB::BYTES, LDS = 2 * BUF;
    static constexpr int KB = DA::KB, KIND = 2;
    static constexpr bool F16 = F16_, OUT_BF16 = OUT_BF16_, LOW = F16, SCORES = DA::KC && DB::KC;   // bf16 results: one accumulator will do
    static_assert(DA::KB == DB::KB, "");
};
struct Straight { static __host__ __device__ constexpr int tile_index(int r) { return r; } };

// the part of its tile that a wave has: WM x WN blocks of 16 x 16 from block (wm WM, wn WN) on
template <class C>
struct Waves {
    static constexpr int ROWS = C::NT / 128, WM = C::TM / 16 / ROWS, WN = C::TN / 32;
    static __device__ __forceinline__ int m(int wave) { return wave % ROWS; }
    static __device__ __forceinline__ int n(int wave) { return wave / ROWS; }
};

// every wave's LDS accesses are done, and its loads from memory still on their way
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A tile's results: stored, and (the scores' product) the statistics of its rows.
template <class C, class LA, class LB, class ACC, class LOW>
__device__ __forceinline__ void finish(const GemmArgs& g, int tm, int tn, int sp, const ACC& acc, const LOW& low) {
    constexpr int WM = Waves<C>::WM, WN = Waves<C>::WN;
    constexpr bool TWO = C::LOW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, h = lane >> 4, wm = Waves<C>::m(wave), wn = Waves<C>::n(wave);
    const float f = g.scale * (g.splits == 1 && g.f0 ? factor_of(g.f0, g.f1, g.f2) : 1.f);
    constexpr bool PAIR = LB::tile_index(16) == 1;               // a lane's blocks j and j + 1 hold neighbouring columns
    auto value = [&](int i, int j, int r) {
        float v = acc[i][j][r];
        if constexpr (TWO) v = C::F16 ? fmaf(low[i][j][r], 0x1p-11f, v) : v + low[i][j][r];
        return v * f;
    };
    // columns n, n + 1 of row m: g.b.rows is even, or the row goes on
    auto put_pair = [&](int64_t m, int64_t n, float a, float b) {
        if (m >= g.a.rows || n >= g.b.rows) return;
        if (!C::SCORES && g.live && !(g.live[m] > 0.f)) a = b = 0.f;
        if (C::OUT_BF16 && g.splits == 1) *(uint32_t*)((uint16_t*)g.out + m * g.ldo + n) = f32_to_bf16_bits(a) | f32_to_bf16_bits(b) << 16;
        else *(v2f*)((float*)g.out + sp * g.slab + m * g.ldo + n) = v2f{a, b};
    };
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; j += PAIR ? 2 : 1) {
            const int64_t n = (int64_t)tn * C::TN + LB::tile_index((wn * WN + j) * 16 + l15);
            if constexpr (PAIR) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t m = (int64_t)tm * C::TM + LA::tile_index((wm * WM + i) * 16 + 4 * h + r);
                    put_pair(m, n, value(i, j, r), value(i, j + 1, r));
                }
            } else {
                // two rows at a time, so that a lane stores two neighbouring columns: an even lane takes row r with its neighbour's
                // column, an odd one row r + 1
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float x = value(i, j, r), y = value(i, j, r + 1);
                    const float px = __int_as_float(dpp16<0xB1>(__float_as_int(x))), py = __int_as_float(dpp16<0xB1>(__float_as_int(y)));
                    const bool odd = lane & 1;
                    const int64_t m = (int64_t)tm * C::TM + LA::tile_index((wm * WM + i) * 16 + 4 * h + r) + (odd ? 1 : 0);
                    put_pair(m, odd ? n - 1 : n, odd ? py : x, odd ? y : px);
                }
            }
        }
    if constexpr (C::SCORES)
        if (g.seg) {
            // the logits are written; this wave's WN * 16 columns of each row: maximum, sum of exp, first column of the maximum
            const float inv = __fdiv_rn(1.f, g.f2[0]);
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t m = (int64_t)tm * C::TM + (wm * WM + i) * 16 + 4 * h + r;
                    float z[WN], mx = -INFINITY, se = 0.f;
                    int am = INT32_MAX;
#pragma unroll
                    for (int j = 0; j < WN; ++j) {
                        const int64_t n = (int64_t)tn * C::TN + (wn * WN + j) * 16 + l15;
                        z[j] = n < g.b.rows ? logit(value(i, j, r), inv) : -INFINITY;
                        if (z[j] > mx) { mx = z[j]; am = (int)n; }
                        if (z[j] != z[j]) se = z[j];             // a NaN stays one whatever the maximum is
                    }
                    const float top = max16(mx);
                    am = min16(mx == top ? am : INT32_MAX);
                    if (top > -INFINITY)
#pragma unroll
                        for (int j = 0; j < WN; ++j) se += exp_neg(z[j] - top);
                    se = sum16(se);
                    if (l15 == 0 && m < g.a.rows) *(v4f*)(g.seg + (m * g.segs + tn * 2 + wn) * 4) = v4f{top, se, __int_as_float(am), 0.f};
                }
        }
}

// what every form of the product starts with: its tile, its part of k, its accumulators
#define GEMM_BEGIN(STAGE_VALUES) \
    constexpr int WM = Waves<C>::WM, WN = Waves<C>::WN, STAGE = STAGE_VALUES; \
    constexpr bool TWO = C::LOW; \
    typedef typename std::conditional<C::F16, v8h, v8bf>::type frag_t; \
    const int per = g.nm * g.nn, sp = item / per, inner = item % per, tn = inner / g.nm, tm = inner % g.nm; \
    const int64_t k0 = sp * g.kstep, k1 = min(g.k, k0 + g.kstep); \
    const int ns = (int)((k1 - k0 + STAGE - 1) / STAGE); \
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = Waves<C>::m(wave), wn = Waves<C>::n(wave); \
    v4f acc[WM][WN], low[TWO ? WM : 1][TWO ? WN : 1]; \
    _Pragma("unroll") for (int i = 0; i < WM; ++i) \
        _Pragma("unroll") for (int j = 0; j < WN; ++j) { \
            acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f}; \
            if constexpr (TWO) low[i][j] = v4f{0.f, 0.f, 0.f, 0.f}; \
        }

template <class C, class F>
__device__ __forceinline__ void mfma(v4f& c, const F& a, const F& b) {
    if constexpr (C::F16) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <class C>
__device__ __forceinline__ bool gemm_tile(const GemmArgs& g, int item, char* smem) {
    GEMM_BEGIN(32)
    constexpr int BUF = C::LDS / C::LBUF, LB0 = C::PA * C::TM * 64, UA = C::LA::UNITS, UNITS = UA + C::LB::UNITS;
    const int l15 = lane & 15, h = lane >> 4;
    typename C::LA A;
    typename C::LB B;
    A.init(g.a, (int64_t)tm * C::TM, threadIdx.x);
    B.init(g.b, (int64_t)tn * C::TN, threadIdx.x);
    const int nfull = (int)((k1 - k0) / STAGE);
    auto fetch = [&](int d, int st) {
        const int64_t k = k0 + (int64_t)st * STAGE;
        if (st < nfull) {
            A.template load<false>(d, g.a, k, k1);
            B.template load<false>(d, g.b, k, k1);
        } else if (st < ns) {
            A.template load<true>(d, g.a, k, k1);
            B.template load<true>(d, g.b, k, k1);
        }
    };
    auto store = [&](int d, int u0, int u1, char* to) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
            if (u >= u0 && u < u1) {
                if (u < UA) A.store(d, u, to);
                else B.store(d, u - UA, to + LB0);
            }
    };
#pragma unroll
    for (int d = 0; d < C::DEPTH; ++d) fetch(d, d);
    if (C::LBUF == 2 && ns) {
        store(0, 0, UNITS, smem);
        fetch(0, C::DEPTH);
    }
    for (int s0 = 0; s0 < ns; s0 += C::DEPTH) {
#pragma unroll
        for (int d = 0; d < C::DEPTH; ++d) {
            const int st = s0 + d, next = (d + 1) % C::DEPTH;
            if (st >= ns) break;
            char* la = smem + (C::LBUF == 2 ? (st & 1) * BUF : 0);
            char* other = smem + (C::LBUF == 2 ? (~st & 1) * BUF : 0);
            if constexpr (C::LBUF == 1) {
                store(d, 0, UNITS, la);
                lds_barrier();
                fetch(d, st + C::DEPTH);
            } else lds_barrier();
            frag_t fb[WN][C::PB];
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int p = 0; p < C::PB; ++p) fb[j][p] = *(const frag_t*)(la + LB0 + lds_at<C::TN>(p, (wn * WN + j) * 16 + l15, h));
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                frag_t fa[C::PA];
#pragma unroll
                for (int p = 0; p < C::PA; ++p) fa[p] = *(const frag_t*)(la + lds_at<C::TM>(p, (wm * WM + i) * 16 + l15, h));
#pragma unroll
                for (int pa = 0; pa < C::PA; ++pa)
#pragma unroll
                    for (int pb = 0; pb < C::PB; ++pb)
                        if (pa + pb < C::KEEP)
#pragma unroll
                            for (int j = 0; j < WN; ++j) mfma<C>(pa + pb == 0 ? acc[i][j] : low[TWO ? i : 0][TWO ? j : 0], fa[pa], fb[j][pb]);
                if constexpr (C::LBUF == 2) {                    // (past the last stage: into a buffer that nothing reads)
                    const int step = i - C::FROM, steps = WM - C::FROM;
                    if (C::FROM > 0 && step == 0) {
                        __builtin_amdgcn_sched_barrier(0);
                        A.pin(next);
                        B.pin(next);
                    }
                    if (step >= 0) store(next, step * UNITS / steps, (step + 1) * UNITS / steps, other);
                }
            }
            if constexpr (C::LBUF == 1) lds_barrier();
            else fetch(next, st + 1 + C::DEPTH);
        }
    }
    finish<C, typename C::LA, typename C::LB>(g, tm, tn, sp, acc, low);
    return false;
}

// A's values are on their way into one LDS buffer, and B's of the next stage go there from registers, while the other is multiplied.  A wave
// waits for A's by count: what it issues after them are the LOADS of B's stage further on.  A's rows go on with zeros to a whole stage, so
// that B's values past the end only have to be numbers wherever the row's (the last storage row's) own are: no load needs a branch, and
// the compiler counts what is on its way.  (Past the last stage it is brought again, into buffers that nothing reads.)
template <class C>
__device__ __forceinline__ bool gemm_mix(const GemmArgs& g, int item, char* smem) {
    GEMM_BEGIN(32)
    constexpr int UNITS = C::LB::UNITS, STEPS = WM - C::FROM;
    const int l15 = lane & 15, h = lane >> 4;
    typename C::DA A;
    typename C::LB B;
    A.init(g.a, (int64_t)tm * C::TM, threadIdx.x);
    B.init(g.b, (int64_t)tn * C::TN, threadIdx.x);
    const int64_t last = k0 + (int64_t)(ns - 1) * STAGE;
    auto bring = [&](int st) {
        A.issue(g.a, min(k0 + (int64_t)st * STAGE, last), smem + (st & 1) * C::BUF);
        asm volatile("" ::: "memory");                            // nothing that is written after it is issued before it
        __builtin_amdgcn_sched_barrier(0);
    };
    auto fetch = [&](int st) {
        B.load_held(0, g.b, k0 + (int64_t)st * STAGE, k1);
        asm volatile("" ::: "memory");
    };
    bring(0);
    fetch(0);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) B.store(0, u, smem + C::DA::BYTES);
    fetch(1);
    for (int st = 0; st < ns; ++st) {                             // (a way out inside, and the compiler would have to count for both)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::LB::LOADS) : "memory");
        lds_barrier();
        bring(st + 1);
        const char* la = smem + (st & 1) * C::BUF;
        const char* lb = la + C::DA::BYTES;
        char* other = smem + (~st & 1) * C::BUF + C::DA::BYTES;
        frag_t fb[WN][C::PB];
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int p = 0; p < C::PB; ++p) fb[j][p] = *(const frag_t*)(lb + lds_at<C::TN>(p, (wn * WN + j) * 16 + l15, h));
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            frag_t fa[C::PA][1];
#pragma unroll
            for (int p = 0; p < C::PA; ++p) C::DA::frags(fa[p], la, p, wm * WM + i, lane);
#pragma unroll
            for (int pa = 0; pa < C::PA; ++pa)
#pragma unroll
                for (int pb = 0; pb < C::PB; ++pb)
                    if (pa + pb < C::KEEP)
#pragma unroll
                        for (int j = 0; j < WN; ++j) mfma<C>(pa + pb == 0 ? acc[i][j] : low[i][j], fa[pa][0], fb[j][pb]);
            const int step = i - C::FROM;                        // (past the last stage: into a buffer that nothing reads)
            if (C::FROM > 0 && step == 0) {
                __builtin_amdgcn_sched_barrier(0);
                B.pin(0);
            }
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                if (step >= 0 && u >= step * UNITS / STEPS && u < (step + 1) * UNITS / STEPS) B.store(0, u, other);
        }
        __builtin_amdgcn_sched_barrier(0);
        fetch(st + 2);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // nothing on its way to LDS when the workgroup ends
    finish<C, Straight, typename C::LB>(g, tm, tn, sp, acc, low);
    return B.outside();
}

// A stage is on its way into one LDS buffer while the other is multiplied, and no register holds it in between.  512 x 16384 x 3584 in
// bf16: scores 69 to 72 us, gradients 127 to 132 us (0.86 and 1.0 PFLOP/s; a large product of a library 1.38).  Measured and left: a third buffer (one
// workgroup a CU less: 112 and 159 us), wave tiles of 128 x 64, one wave a SIMD, with the fragments' reads and the loads spread among the
// MFMAs by hand (4 % of the scores' time), and the loads alone spread (slower).  What bounds it: MFMAs are busy 46 to 51 % of the clocks; the
// waves wait 28 % of theirs for a stage, whose loads have the one before to arrive in, and 38 % for their turn to issue.
template <class C>
__device__ __forceinline__ bool gemm_straight(const GemmArgs& g, int item, char* smem) {
    GEMM_BEGIN(C::KB * 32)
    typename C::DA A;
    typename C::DB B;
    A.init(g.a, (int64_t)tm * C::TM, threadIdx.x);
    B.init(g.b, (int64_t)tn * C::TN, threadIdx.x);
    const int nfull = (int)((k1 - k0) / STAGE);
    auto bring = [&](int st, int buf) {
        char* la = smem + buf * C::BUF;
        const int64_t k = k0 + (int64_t)st * STAGE;
        if (st < nfull) {
            A.issue(g.a, k, la);
            B.issue(g.b, k, la + C::DA::BYTES);
        } else if (st < ns) {
            A.tail(g.a, k, k1, la);
            B.tail(g.b, k, k1, la + C::DA::BYTES);
        }
    };
    bring(0, 0);
    for (int st = 0; st < ns; ++st) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        bring(st + 1, (st + 1) & 1);   // into the buffer that every wave has done with
        const char* la = smem + (st & 1) * C::BUF;
        const char* lb = la + C::DA::BYTES;
#pragma unroll
        for (int kb = 0; kb < C::KB; ++kb) {
            frag_t fa[C::PA][WM], fb[C::PB][WN];
#pragma unroll
            for (int p = 0; p < C::PB; ++p) C::DB::frags(fb[p], lb, p + kb, wn * WN, lane);
#pragma unroll
            for (int pa = 0; pa < C::PA; ++pa) {
                C::DA::frags(fa[pa], la, pa + kb, wm * WM, lane);
#pragma unroll
                for (int i = 0; i < WM; ++i)
#pragma unroll
                    for (int pb = 0; pb < C::PB; ++pb)
                        if (pa + pb < C::KEEP)
#pragma unroll
                            for (int j = 0; j < WN; ++j) mfma<C>(!TWO || pa + pb == 0 ? acc[i][j] : low[TWO ? i : 0][TWO ? j : 0], fa[pa][i], fb[pb][j]);
            }
        }
    }
    finish<C, Straight, Straight>(g, tm, tn, sp, acc, low);
    return false;
}
template <class C>
__device__ __forceinline__ bool gemm_any(const GemmArgs& g, int item, char* smem) {
    if constexpr (C::KIND == 0) return gemm_tile<C>(g, item, smem);
    else if constexpr (C::KIND == 1) return gemm_mix<C>(g, item, smem);
    else return gemm_straight<C>(g, item, smem);
}

// an XCD (every eighth id) takes a run of neighbouring tiles: of one part of k, one n tile's next to each other, so that both operands'
// values of that part are fetched into one L2 or two (512 x 16384 x 3584 in bf16, a step: 251 us; with an n tile's parts of k next to each
// other every L2 fetched all of g for each of its n tiles, 0.7 GB in all: 261 us)
__device__ __forceinline__ int item_of(int id, int n) { return (id & 7) * ((n + 7) >> 3) + (id >> 3); }

// flag: null, or the word that says whether the fp16 parts hold the values; the launch runs where it equals run_if
template <class C>
__global__ __launch_bounds__(C::NT, 2) void distill_scores_kernel(const GemmArgs g, const unsigned* flag, unsigned run_if, unsigned* raise,
                                                                const unsigned* rows_out, int64_t nrows_out, unsigned* clear, int nclear) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    if (flag && *flag != run_if) return;
    if (clear && blockIdx.x == 0)                                 // the arrival counters of the next launch
        for (int i = threadIdx.x; i < nclear; i += C::NT) clear[i] = 0u;
    const int n = g.nn * g.nm * g.splits, item = item_of(blockIdx.x, n);
    bool bad = false;
    if (raise && blockIdx.x == 0)
        for (int64_t i = threadIdx.x; i < nrows_out; i += C::NT) bad |= rows_out[i] != 0u;
    if (item < n) bad |= gemm_any<C>(g, item, smem_raw);
    if (raise && bad) __hip_atomic_store(raise, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// both gradients' products in one launch: the first n0 workgroups (a multiple of 8) take dq
template <class CQ, class CP>
__global__ __launch_bounds__(CQ::NT, 2) void distill_grads_kernel(const GemmArgs gq, const GemmArgs gp, int n0, const unsigned* flag, unsigned run_if) {
    static_assert(CQ::NT == CP::NT, "");
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    if (flag && *flag != run_if) return;
    if ((int)blockIdx.x < n0) {
        const int n = gq.nn * gq.nm * gq.splits, item = item_of(blockIdx.x, n);
        if (item < n) gemm_any<CQ>(gq, item, smem_raw);
    } else {
        const int n = gp.nn * gp.nm * gp.splits, item = item_of(blockIdx.x - n0, n);
        if (item < n) gemm_any<CP>(gp, item, smem_raw);
    }
}

// whether entry (index, score) of a list is one
__device__ __forceinline__ bool is_entry(int64_t j, float x) { return j >= 0 && !(x == -INFINITY); }

// the queries' fp16 parts, once for all tiles of the two products that read them, zeros for a row without an entry; rows_out[b]: row b does
// not fit them.  dpad: d up to 32s
__global__ __launch_bounds__(256) void distill_split_kernel(const float* __restrict__ q, int d, int dpad, const int64_t* __restrict__ idx,
                                                            const float* __restrict__ score, int list, char* __restrict__ out,
                                                            unsigned* __restrict__ rows_out, unsigned* __restrict__ flag) {
    __shared__ float red[4];
    const int64_t b = blockIdx.x;
    if (b == 0 && threadIdx.x == 0) *flag = 0u;
    bool some = false;
    for (int i = threadIdx.x; i < list; i += 256) some |= is_entry(idx[b * list + i], score[b * list + i]);
    some = __syncthreads_or(some);
    float top = 0.f;
    for (int k = threadIdx.x * 4; k < dpad; k += 1024) {
        const v4f x = k < d && some ? *(const v4f*)(q + b * d + k) : v4f{0.f, 0.f, 0.f, 0.f};
        uint32_t lo[2], hi[2];
        split_pair(x[0], x[1], lo);
        split_pair(x[2], x[3], hi);
        char* to = out + b * dpad * 4 + split_at(k);
        *(uint2*)to = uint2{lo[0], hi[0]};
        *(uint2*)(to + 64) = uint2{lo[1], hi[1]};
#pragma unroll
        for (int c = 0; c < 4; ++c) top = fmaxf(top, fabsf(x[c]));
    }
    for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        rows_out[b] = top > 0.f && !(top >= H_MIN && top <= H_LOW) ? 1u : 0u;
    }
}

// ---- the rows: logsumexp, the teacher's list, the loss -------------------------------------------------------------------
// A workgroup a row where the product left its waves' statistics (two records a tile: 106 for 5000 columns, 256 for 16 384), else one for 2048 columns, which adds up the
// slabs, and the last of a row's goes on.  Bound by latency: records, list, the list's logits, five reductions, two arrivals, one after
// another.  1000 rows of 5000, list of 10: 14 us; 512 of 16 384, list of 100: 16.5; 128 of 1024 in 8 slabs, list of 64: 11.
struct RowArgs {
    const float* part;               // slabs [splits][B][lds] of s
    float* s;                        // their sum (part itself where there is one)
    int splits, segs;
    bool ready;                      // seg is there: one workgroup a row
    int64_t slab, lds;
    const float* temp;
    const int64_t* idx;
    const float* score;
    float teacher_temp;
    int64_t B, T;
    int k;
    float* seg;                      // [B][segs][4]: maximum, sum of exp(z - maximum), its first column, 1 where a z is NaN
    float* norm;                     // [B] the row's maximum, then [B] 1 / its sum of exp(z - maximum)
    float* t;                        // [B][k]: the teacher's share of column li (all of a column's entries at the first of them), or 0
    int* li;                         // [B][k]: the column, -1 = nothing
    float* row;                      // [B] row losses, then [B] agreement, then [B] 1 where the row has an entry
    float* stat;                     // [0]: 1 / rows that have an entry
    unsigned* cnt;                   // [B] segments that have arrived, [1] groups of 32 rows, [groups] their rows
    float* out_loss;
    float* out_agree;
};

// Values handed to another workgroup of the same launch: stored and loaded past the caches that are not common to the chip.
__device__ __forceinline__ void put(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float get(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// Whether this workgroup is the last of n to arrive; its thread 0 made the put()s that the last one get()s.
__device__ __forceinline__ bool arrive_last(unsigned* cnt, unsigned n, unsigned* flag) {
    if (threadIdx.x == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the puts have reached the chip's common memory before the arrival counts
        *flag = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1 ? 1u : 0u;
    }
    __syncthreads();
    return *flag != 0u;
}

struct Red { float a, b; int c; };
// maximum, sum and minimum over the workgroup of 256 threads, in one round; fixed order
__device__ __forceinline__ Red block_red(float mx, float sum, int mn, Red* red) {
    mx = max16(mx);
    sum = sum16(sum);
    mn = min16(mn);
#pragma unroll
    for (int m = 16; m < 64; m <<= 1) {
        mx = fmaxf(mx, __shfl_xor(mx, m, 64));
        sum += __shfl_xor(sum, m, 64);
        mn = min(mn, __shfl_xor(mn, m, 64));
    }
    __syncthreads();                                             // the last round has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = Red{mx, sum, mn};
    __syncthreads();
    Red r = red[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) { r.a = fmaxf(r.a, red[w].a); r.b += red[w].b; r.c = min(r.c, red[w].c); }
    return r;
}
// three sums over the workgroup at once
__device__ __forceinline__ void block_sum(float& x, float& y, int& n, Red* red) {
    x = sum16(x);
    y = sum16(y);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        if (m >= 16) { x += __shfl_xor(x, m, 64); y += __shfl_xor(y, m, 64); }
        n += __shfl_xor(n, m, 64);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = Red{x, y, n};
    __syncthreads();
    x = (red[0].a + red[1].a) + (red[2].a + red[3].a);
    y = (red[0].b + red[1].b) + (red[2].b + red[3].b);
    n = (red[0].c + red[1].c) + (red[2].c + red[3].c);
}

__global__ __launch_bounds__(256) void distill_row_kernel(const RowArgs a) {
    __shared__ Red red[4];
    __shared__ __attribute__((aligned(16))) float le[DISTILL_MAX_K];
    __shared__ __attribute__((aligned(16))) int li[DISTILL_MAX_K];
    __shared__ unsigned last;
    const int64_t b = blockIdx.y;
    const int tid = threadIdx.x;
    const float inv = __fdiv_rn(1.f, a.temp[0]);
    const float* part = a.part + b * a.lds;
    // ---- this segment's columns: the slabs' sum, the maximum of z and its first column, the sum of exp
    float mx, se;
    int am;
    bool nan = false;
    // the teacher's list: entries at[], scores v[], logits z[]; best: the largest score, bad: an entry that makes the row NaN
    const int64_t* idx = a.idx + b * a.k;
    const float* score = a.score + b * a.k;
    float v[4], z[4], best = -INFINITY, bad = 0.f;
    int at[4], some = 0;
    auto take_list = [&] {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = tid + u * 256;
            at[u] = -1;
            v[u] = -INFINITY;
            if (i >= a.k) continue;
            const int64_t j = idx[i];
            const float x = score[i];
            if (is_entry(j, x)) {
                some = 1;
                if (j >= a.T || !(x < INFINITY)) bad = 1.f;      // a column that is not there, a score that is no number: the row is NaN
                else { at[u] = (int)j; v[u] = x; best = fmaxf(best, x); }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            z[u] = 0.f;
            if (at[u] >= 0)
                for (int p = 0; p < a.splits; ++p) z[u] += part[p * a.slab + at[u]];
        }
    };
    if (!a.ready) {
        const int64_t j0 = (int64_t)blockIdx.x * DISTILL_SEG + tid * 4;
        v4f x[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
        bool in[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) in[u] = j0 + u * 1024 < a.T;
        for (int p = 0; p < a.splits; p += 4) {                   // four slabs' loads in flight; slabs in order
            v4f y[4][2];
#pragma unroll
            for (int o = 0; o < 4; ++o)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (p + o < a.splits && in[u]) y[o][u] = *(const v4f*)(part + (p + o) * a.slab + j0 + u * 1024);
#pragma unroll
            for (int o = 0; o < 4; ++o)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (p + o < a.splits && in[u]) x[u] += y[o][u];
        }
        mx = -INFINITY;
        am = INT32_MAX;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!in[u]) continue;
            if (a.splits > 1) *(v4f*)(a.s + b * a.lds + j0 + u * 1024) = x[u];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (j0 + u * 1024 + c >= a.T) { x[u][c] = -INFINITY; continue; }
                x[u][c] = logit(x[u][c], inv);
                if (x[u][c] > mx) { mx = x[u][c]; am = (int)(j0 + u * 1024 + c); }
                nan |= x[u][c] != x[u][c];
            }
        }
        const float mine = mx;
        const Red r = block_red(mx, 0.f, 0, red);
        mx = r.a;
        se = 0.f;
        if (mx > -INFINITY)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (in[u])
#pragma unroll
                    for (int c = 0; c < 4; ++c) se += exp_neg(x[u][c] - mx);
        const Red r2 = block_red(nan ? 1.f : 0.f, se, mine == mx && mx > -INFINITY ? am : INT32_MAX, red);
        nan = r2.a > 0.f;
        se = r2.b;
        am = r2.c;
    }
    if (a.ready) {
        // ---- the product's waves have left a record for each of their stretches of the row
        const v4f* seg = (const v4f*)a.seg + b * a.segs;
        const v4f first = tid < a.segs ? seg[tid] : v4f{-INFINITY, 0.f, __int_as_float(INT32_MAX), 0.f};
        take_list();                                             // (its loads run beside the records')
        mx = first[0];
        for (int i = tid + 256; i < a.segs; i += 256) mx = fmaxf(mx, seg[i][0]);
        mx = block_red(mx, 0.f, 0, red).a;
        se = 0.f;
        am = INT32_MAX;
        for (int i = tid; i < a.segs; i += 256) {
            const v4f x = i == tid ? first : seg[i];
            if (x[0] == mx) am = min(am, __float_as_int(x[2]));
            se += x[0] > -INFINITY ? x[1] * exp_neg(x[0] - mx) : x[1];   // (nothing but NaN there: x[1] is NaN, else 0)
        }
        const Red r = block_red(0.f, se, am, red);
        se = r.b;
        am = r.c;
    } else if (a.segs > 1) {
        float* seg = a.seg + b * a.segs * 4;
        if (tid == 0) {
            put(seg + blockIdx.x * 4, mx);
            put(seg + blockIdx.x * 4 + 1, se);
            put(seg + blockIdx.x * 4 + 2, __int_as_float(am));
            put(seg + blockIdx.x * 4 + 3, nan ? 1.f : 0.f);
        }
        if (!arrive_last(a.cnt + b, (unsigned)a.segs, &last)) return;
        // ---- the last segment of the row: all of them together
        mx = -INFINITY;
        float any = 0.f;
        for (int i = tid; i < a.segs; i += 256) { mx = fmaxf(mx, get(seg + i * 4)); any = fmaxf(any, get(seg + i * 4 + 3)); }
        const Red r = block_red(mx, any, 0, red);
        mx = r.a;
        nan = r.b > 0.f;
        se = 0.f;
        am = INT32_MAX;
        if (mx > -INFINITY)
            for (int i = tid; i < a.segs; i += 256) {
                const float m = get(seg + i * 4);
                if (m > -INFINITY) se += get(seg + i * 4 + 1) * exp_neg(m - mx);
                if (m == mx) am = min(am, __float_as_int(get(seg + i * 4 + 2)));
            }
        const Red r2 = block_red(0.f, se, am, red);
        se = r2.b;
        am = r2.c;
    }
    if (nan) se = __uint_as_float(0x7FC00000u);
    // ---- the teacher's list: softmax over its entries, the best of them, the row's loss
    if (!a.ready) take_list();
    const int k8 = (a.k + 7) & ~7;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (tid + u * 256 < k8) li[tid + u * 256] = at[u];       // (-1 past the list)
    {
        const Red r = block_red(best, bad, -some, red);
        best = r.a;
        bad = r.b;
        some = -r.c;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = logit(z[u], inv) - mx;
    float e[4], esum = 0.f;
    int first = INT32_MAX;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = tid + u * 256;
        e[u] = 0.f;
        const bool top = v[u] == best;                           // (of the scores: a quotient by a large temperature may be 0 for others too)
        v[u] = __fdiv_rn(v[u] - best, a.teacher_temp);
        if (at[u] >= 0) {
            e[u] = exp_neg(v[u]);
            if (top) first = min(first, i);
        }
        esum += e[u];
        if (i < k8) le[i] = e[u];
    }
    {
        const Red r = block_red(0.f, esum, first, red);
        esum = r.b;
        first = r.c;
    }
    const float loge = logf(esum);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = tid + u * 256;
        if (i >= a.k) continue;
        const float p = bad == 0.f && at[u] >= 0 ? __fdiv_rn(e[u], esum) : 0.f;
        if (p > 0.f) sum += p * ((v[u] - loge) - z[u]);
        // a column's shares together, at its first entry
        float all = 0.f;
        bool mine = at[u] >= 0 && bad == 0.f;
        if (mine)
            for (int o = 0; o < k8; o += 8) {                    // eight at a time: their reads are one wait
                int4 l[2];
                v4f w[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) { l[h] = *(const int4*)(li + o + 4 * h); w[h] = *(const v4f*)(le + o + 4 * h); }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int lo[4] = {l[h].x, l[h].y, l[h].z, l[h].w};
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (lo[c] == at[u]) { mine = mine && o + 4 * h + c >= i; all += w[h][c]; }
                }
            }
        a.t[b * a.k + i] = mine ? __fdiv_rn(all, esum) : 0.f;
        a.li[b * a.k + i] = mine ? at[u] : -1;
    }
    sum = block_red(0.f, sum, 0, red).b;
    if (bad > 0.f) se = __uint_as_float(0x7FC00000u);
    if (tid == 0) {
        a.norm[b] = mx;
        a.norm[a.B + b] = __fdiv_rn(1.f, se);
        put(a.row + b, some ? sum + logf(se) : 0.f);
        put(a.row + a.B + b, some && bad == 0.f && am == li[first] ? 1.f : 0.f);
        put(a.row + 2 * a.B + b, some ? 1.f : 0.f);
    }
    // 32 rows arrive on a counter of theirs, the last of them on the common one (arrivals on one word follow each other some 40 ns apart)
    const int64_t group = b / 32, groups = (a.B + 31) / 32;
    if (!arrive_last(a.cnt + a.B + 1 + group, (unsigned)min((int64_t)32, a.B - group * 32), &last)) return;
    __syncthreads();
    if (!arrive_last(a.cnt + a.B, (unsigned)groups, &last)) return;
    // ---- the last row: the means
    float ls = 0.f, hs = 0.f;
    int ns = 0;
    for (int64_t i = tid; i < a.B; i += 256) {
        ls += get(a.row + i);
        hs += get(a.row + a.B + i);
        ns += get(a.row + 2 * a.B + i) > 0.f ? 1 : 0;
    }
    block_sum(ls, hs, ns, red);
    const float n = fmaxf((float)ns, 1.f);
    if (tid == 0) {
        a.out_loss[0] = __fdiv_rn(ls, n);
        a.out_agree[0] = __fdiv_rn(hs, n);
        a.stat[0] = __fdiv_rn(1.f, n);
    }
}

// ---- softmax - target ----------------------------------------------------------------------------------------------------
// HBM-bound: the logits once, g once, in the form that the products take (512 x 16 384: 67 MB in 16.5 us).  One workgroup more a row copies its
// query for the candidates' product (1.2 us of them, 7 MB).
enum { G_F32, G_F16, G_BF16 };
struct GradArgs {
    const float* s;                  // [B][lds]
    int64_t lds;
    const float* norm;               // [2][rows]
    const float* t;
    const int* li;
    const float* has;                // [B]: 1 where the row has an entry
    const float* temp;
    int64_t T, ldg;
    int k;
    int form;                        // G_F32, G_F16 (G_F32 where flag is set) or G_BF16
    const unsigned* flag;
    void* g;                         // [B][ldg] fp32 or two parts of 16 bits; zeros from T on
    int segs, seg0;                  // seg0: this launch's first
    float* dt;                       // [B][segs]: sums of (softmax - target) z
    const char* q;
    char* qlive;                     // given (segs + 1 workgroups a row): the queries, zeros for rows without an entry.  G_F16: where flag is set
    int qbytes;                      // a query's
};

__global__ __launch_bounds__(256) void distill_grad_kernel(const GradArgs a) {
    __shared__ __attribute__((aligned(16))) float target[DISTILL_SEG];
    __shared__ Red red[4];
    const int seg = a.seg0 + (int)blockIdx.x;
    const int64_t b = blockIdx.y, j0 = (int64_t)seg * DISTILL_SEG;
    const int tid = threadIdx.x;
    const bool has = a.has[b] > 0.f;
    const int form = a.form == G_F16 && *a.flag ? G_F32 : a.form;
    if (seg == a.segs) {
        if (form == G_F16) return;                               // (the split kernel has seen to their parts)
        for (int i = tid * 16; i < a.qbytes; i += 4096)
            *(v4u*)(a.qlive + b * a.qbytes + i) = has ? *(const v4u*)(a.q + b * a.qbytes + i) : v4u{0, 0, 0, 0};
        return;
    }
    const float inv = __fdiv_rn(1.f, a.temp[0]), mx = a.norm[b], one = a.norm[gridDim.y + b];
    v4f x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (j0 + tid * 4 + u * 1024 < a.ldg) x[u] = *(const v4f*)(a.s + b * a.lds + j0 + tid * 4 + u * 1024);   // ldg columns are there in s too
#pragma unroll
    for (int u = 0; u < 2; ++u) *(v4f*)(target + tid * 4 + u * 1024) = v4f{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    if (has)
        for (int i = tid; i < a.k; i += 256) {
            const int at = a.li[b * a.k + i];                    // no column twice
            if (at >= j0 && at < j0 + DISTILL_SEG) target[at - j0] = a.t[b * a.k + i];
        }
    __syncthreads();
    float dt = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t j = j0 + tid * 4 + u * 1024;
        if (j >= a.ldg) continue;
        const v4f tg = *(const v4f*)(target + tid * 4 + u * 1024);
        v4f y;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float z = logit(x[u][c], inv);
            y[c] = j + c < a.T && has ? fmaf(exp_neg(z - mx), one, -tg[c]) : 0.f;
            if (j + c < a.T && has) dt += y[c] * z;
        }
        if (form == G_F32) *(v4f*)((float*)a.g + b * a.ldg + j) = y;
        else {
            uint32_t lo[2], hi[2];
            if (form == G_F16) {
                split_pair(y[0] * G_SCALE, y[1] * G_SCALE, lo);
                split_pair(y[2] * G_SCALE, y[3] * G_SCALE, hi);
            } else {
                split_round(y[0], y[1], lo);
                split_round(y[2], y[3], hi);
            }
            char* out = (char*)a.g + b * a.ldg * 4 + split_at(j);
            *(uint2*)out = uint2{lo[0], hi[0]};
            *(uint2*)(out + 64) = uint2{lo[1], hi[1]};
        }
    }
    dt = block_red(0.f, dt, 0, red).b;
    if (tid == 0) a.dt[b * a.segs + seg] = dt;
}

// ---- sums of the split products' slabs, and of the temperature's gradient ------------------------------------------------
struct SumArgs {
    const float* part[2];
    void* out[2];
    int64_t n[2];                    // values, a multiple of 4 (0: nothing to do)
    int splits[2];
    int blocks0;                     // workgroups of the first
    const float* live;               // of the first's rows of d values: one that is not above 0 gives zeros
    int d;
    const float* dt;
    int64_t ndt;
    const float *f0, *f1, *f2;       // grad_out, 1 / rows, temp
    float* d_temp;                   // null: not wanted
};

template <bool BF16>
__global__ __launch_bounds__(256) void distill_sum_kernel(const SumArgs a) {
    __shared__ Red red[4];
    const float f = factor_of(a.f0, a.f1, a.f2);
    if (blockIdx.x == gridDim.x - 1) {                            // the last workgroup: the temperature
        if (!a.d_temp) return;
        float v = 0.f;
        for (int64_t i = threadIdx.x; i < a.ndt; i += 256) v += a.dt[i];
        v = block_red(0.f, v, 0, red).b;
        if (threadIdx.x == 0) a.d_temp[0] = -v * f;
        return;
    }
    const int which = (int)blockIdx.x >= a.blocks0;
    const int64_t i = ((int64_t)(blockIdx.x - (which ? a.blocks0 : 0)) * 256 + threadIdx.x) * 4;
    if (i >= a.n[which]) return;
    v4f x = v4f{0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < a.splits[which]; p += 4) {
        v4f y[4];
#pragma unroll
        for (int o = 0; o < 4; ++o)
            if (p + o < a.splits[which]) y[o] = *(const v4f*)(a.part[which] + (p + o) * a.n[which] + i);
#pragma unroll
        for (int o = 0; o < 4; ++o)
            if (p + o < a.splits[which]) x += y[o];
    }
    x *= f;
    if (which == 0 && !(a.live[(uint32_t)i / (uint32_t)a.d] > 0.f)) x = v4f{0.f, 0.f, 0.f, 0.f};   // (at most 65 535 x 65 536 values)
    if constexpr (BF16) {
        uint32_t lo = f32_to_bf16_bits(x[0]) | f32_to_bf16_bits(x[1]) << 16, hi = f32_to_bf16_bits(x[2]) | f32_to_bf16_bits(x[3]) << 16;
        *(uint2*)((uint16_t*)a.out[which] + i) = uint2{lo, hi};
    } else *(v4f*)((float*)a.out[which] + i) = x;
}

// ---- plans ---------------------------------------------------------------------------------------------------------------
struct Plan { int tile, splits; int64_t kstep; int nm, nn; };

// Tiles of 128 x 128 (two workgroups a CU) or 64 x 64 (four), and k in so many parts that the CUs have work.  A tile of 128
// needs half the operands' reads; tiles of 64 give more workgroups.  The choice goes by the tiles of 128 times the parts of 8 stages that k has
// (`least`).  Measured, us, 64 / 128:
//   fp32 scores, from 288      128 x 1024 x 4096 (72) 36 / 45, 256 x 4096 x 1024 (192) 38 / 48, 128 x 4096 x 4096 (288) 50 / 50, 256 x 8192 x 1024 (384) 52 / 50
//   fp32 gradients, from 128   by the product with the longer k: 128 x 1024 x 4096 (96) 41 / 47, 1000 x 1000 x 1024 (128) 60 / 53,
//                              256 x 4096 x 1024 (144) 59 / 51, 128 x 4096 x 4096 (288) 100 / 69
//   bf16, from 64              scores of 128 x 1024 x 4096 (72) 30 / 22, 128 x 8192 x 1024 (192) 28 / 24
// Parts of k: until two workgroups a CU (tiles of 64: four) run, as long as a part keeps 8 stages of 64; tiles of 64 until every CU has one, as
// long as it keeps two.  More parts are more slabs to write and add up: 128 x 1024 x 4096, forward 27 us, with parts until four a CU run 35,
// backward 32 and 38; 32 x 21 000 x 4096 221 and, one workgroup a CU, 256; 17 x 300 x 4096, forward 19.2 us with 16 parts, 20.8 with 32 (cap).
#define LEAST_SCORES 288
#define LEAST_GRADS 128
#define LEAST_BF16 64
static int64_t parts_of(const Plan& p, int64_t stages, int cap) {
    const int64_t tiles = (int64_t)p.nm * p.nn;
    int64_t sp = min((p.tile == 128 ? 512 : 1024) / tiles, stages / 8);
    if (p.tile == 64) sp = max(sp, min(256 / tiles, stages / 2));
    return max((int64_t)1, min(sp, (int64_t)cap));
}
static Plan plan(int64_t m, int64_t n, int64_t k, int least, int cap) {
    Plan p;
    auto tiles = [&](int t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
    const int64_t stages = (k + 63) / 64;
    p.tile = m > 64 && n > 64 && tiles(128) * (stages / 8 + 1) >= least ? 128 : 64;
    p.nm = (int)((m + p.tile - 1) / p.tile);
    p.nn = (int)((n + p.tile - 1) / p.tile);
    const int64_t sp = parts_of(p, stages, cap);
    const int64_t per = (stages + sp - 1) / sp;
    p.kstep = per * 64;
    p.splits = (int)((stages + per - 1) / per);
    return p;
}

static inline size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

struct FwdLayout {
    Plan s;
    bool fast;                       // fp32 by fp16 parts
    bool narrow;                     // bf16: tiles of 128 x 96
    int64_t lds;
    int segs;
    size_t off_s, off_seg, off_norm, off_t, off_li, off_row, off_stat, off_cnt, off_q, off_qout, off_flag, total;
};

static FwdLayout fwd_layout(int dtype, int64_t B, int64_t T, int d, int k) {
    FwdLayout L;
    L.s = plan(B, T, d, dtype == ABC_DT_BF16 ? LEAST_BF16 : LEAST_SCORES, 16);
    // bf16, two workgroups a CU: where one round holds tiles of 128 x 96 they fill it better than those of 128 x 128 (1000 x 5000 x 3584, forward: 67 us
    // and 76; 1000 x 6100 x 4096 75 and 85; 256 x 20 000 x 3584 60 and 66; 500 x 7000 x 768 31 and 30), and better than two parts of a short k (1000 x 3200 x
    // 1024 36 and 41, 128 x 30 000 x 1024 32 and 39; but 1000 x 3500 x 3584 59 and 56).
    const int64_t n96 = (T + 95) / 96;
    L.narrow = dtype == ABC_DT_BF16 && L.s.tile == 128 && (L.s.splits == 1 || d < 2048) && L.s.nm * n96 > 256 && L.s.nm * n96 <= 512;
    if (L.narrow) { L.s.nn = (int)n96; L.s.splits = 1; L.s.kstep = (d + 63) / 64 * 64; }
    L.lds = (T + 31) / 32 * 32;
    L.segs = L.s.splits == 1 ? L.s.nn * 2 : (int)((T + DISTILL_SEG - 1) / DISTILL_SEG);
    // From about 8 GFLOP a product on, half the matrix work is worth the launches that find out and then return (256 x 16 384 x 1024, forward and
    // backward: 121 us, without 150).
    L.fast = dtype == ABC_DT_F32 && L.s.tile == 128 && 2.0 * (double)B * (double)T * d >= 8e9;
    // (slabs, which the backward keeps without reading them: 512 tiles of 64 KB, 1024 of 16 KB, 32 MB at most)
    size_t o = up((size_t)L.s.splits * B * L.lds * 4);
    L.off_s = 0;
    if (L.s.splits > 1) { L.off_s = o; o += up((size_t)B * L.lds * 4); }
    L.off_seg = o; o += up((size_t)B * L.segs * 16);
    L.off_norm = o; o += up((size_t)B * 8);
    L.off_t = o; o += up((size_t)B * k * 4);
    L.off_li = o; o += up((size_t)B * k * 4);
    L.off_row = o; o += up((size_t)B * 12);
    L.off_stat = o; o += 256;
    L.off_cnt = o; o += up((size_t)(B + 1 + (B + 31) / 32) * 4);
    L.off_q = o; o += L.fast ? up((size_t)B * ((d + 31) / 32 * 32) * 4) : 0;
    L.off_qout = o; o += L.fast ? up((size_t)B * 4) : 0;
    L.off_flag = o; o += 256;
    L.total = o;
    return L;
}

struct BwdLayout { Plan q, p; int64_t ldg; int segs; size_t off_g, off_dt, off_pq, off_pp, off_ql, total; };
static BwdLayout bwd_layout(int dtype, int64_t B, int64_t C, int64_t T, int d, bool fast, bool dq, bool dp) {
    const int least = dtype == ABC_DT_BF16 ? LEAST_BF16 : LEAST_GRADS;
    BwdLayout L;
    L.ldg = (T + 31) / 32 * 32;                                // as the logits' rows
    L.segs = (int)((L.ldg + DISTILL_SEG - 1) / DISTILL_SEG);
    L.q = plan(B, d, T, least, 32);
    L.p = plan(C, d, B, least, 32);
    if (fast || (L.q.tile == 128) != (L.p.tile == 128)) {         // one launch, one kind of tile: that of the larger product
        const int tile = fast || (T >= B ? L.q.tile : L.p.tile) == 128 ? 128 : 64;
        auto with = [&](Plan& x, int64_t m, int64_t n, int64_t k) {
            if (x.tile == tile) return;
            x.tile = tile;
            x.nm = (int)((m + tile - 1) / tile);
            x.nn = (int)((n + tile - 1) / tile);
            const int64_t stages = (k + 63) / 64, sp = parts_of(x, stages, 32);
            const int64_t per = (stages + sp - 1) / sp;
            x.kstep = per * 64;
            x.splits = (int)((stages + per - 1) / per);
        };
        with(L.q, B, d, T);
        with(L.p, C, d, B);
    }
    size_t o = up((size_t)B * L.ldg * 4);
    L.off_g = 0;
    L.off_dt = o; o += up((size_t)B * L.segs * 4);
    L.off_pq = o; o += dq && L.q.splits > 1 ? up((size_t)L.q.splits * B * d * 4) : 0;
    L.off_pp = o; o += dp && L.p.splits > 1 ? up((size_t)L.p.splits * C * d * 4) : 0;
    L.off_ql = o; o += dp ? up((size_t)B * d * (dtype == ABC_DT_BF16 ? 2 : 4)) : 0;
    L.total = o;
    return L;
}

#define MAX_TILES (1 << 23)           // a launch, of two products' tiles, has fewer than 2^32 threads
static int64_t tiles_of(int64_t rows, int tile) { return (rows + tile - 1) / tile; }

static int distill_check(int dtype, int64_t B, int64_t C, int64_t M, int d, int k) {
    if (dtype != ABC_DT_F32 && dtype != ABC_DT_BF16) return abc_fail_invalid("distill: embeddings must be f32 or bf16");
    if (B < 1 || C < 1 || M < 0) return abc_fail_invalid("distill: need at least one query and one candidate");
    if (B > 65535 || C > 0x7FFFFFF0ll || M > 0x7FFFFFF0ll || C + M > 0x7FFFFFF0ll) return abc_fail_invalid("distill: at most 65535 queries and 2^31 - 16 candidates");
    if (tiles_of(C + M, 64) * tiles_of(B, 64) > MAX_TILES || tiles_of(C, 64) * tiles_of(d, 64) > MAX_TILES)
        return abc_fail_invalid("distill: too many query-candidate pairs for one launch (2^23 tiles of 64 x 64)");
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
    return bwd_layout(dtype, B, C, C + M, d, fwd_layout(dtype, B, C + M, d, k).fast, true, true).total;
}

static GemmArgs gemm_args(const Side& a, const Side& b, int64_t k, const Plan& p, void* out, int64_t ldo, int64_t slab) {
    GemmArgs g = {};
    g.a = a; g.b = b; g.k = k; g.splits = p.splits; g.kstep = p.kstep; g.nm = p.nm; g.nn = p.nn;
    g.out = out; g.ldo = ldo; g.slab = slab; g.scale = 1.f;
    return g;
}
static unsigned groups_of(const GemmArgs& g) { return (unsigned)(((int64_t)g.nn * g.nm * g.splits + 7) / 8 * 8); }

// dynamic LDS past 64 KB has to be asked for, of the current device's copy of the kernel
static void allow_lds(const void* kernel, size_t lds) {
    if (lds > 65536) (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);   // a refusal shows at the launch
}
template <class C>
static void launch_scores(const GemmArgs& g, const unsigned* flag, unsigned run_if, unsigned* raise, const unsigned* rows_out, int64_t B,
                          unsigned* clear, int nclear, hipStream_t st) {
    allow_lds((const void*)distill_scores_kernel<C>, C::LDS);
    hipLaunchKernelGGL((distill_scores_kernel<C>), dim3(groups_of(g)), dim3(C::NT), C::LDS, st, g, flag, run_if, raise, rows_out, B, clear, nclear);
}
template <class CQ, class CP>
static void launch_grads(const GemmArgs& gq, const GemmArgs& gp, bool dq, bool dp, const unsigned* flag, unsigned run_if, hipStream_t st) {
    const unsigned n0 = dq ? groups_of(gq) : 0, n1 = dp ? groups_of(gp) : 0;
    const size_t lds = (size_t)(CQ::LDS > CP::LDS ? CQ::LDS : CP::LDS);
    allow_lds((const void*)distill_grads_kernel<CQ, CP>, lds);
    hipLaunchKernelGGL((distill_grads_kernel<CQ, CP>), dim3(n0 + n1), dim3(CQ::NT), lds, st, gq, gp, (int)n0, flag, run_if);
}

// s: bf16; fp32 by three bf16 parts (128 / 64 wide tiles); fp32 by two fp16 parts (the queries' are ready)
typedef CfgDma<DmaKC<1, 128>, DmaKC<1, 128>, 1, 1, 128, 128, 256, false, false> ScoresB128;
typedef CfgDma<DmaKC<1, 128>, DmaKC<1, 96>, 1, 1, 128, 96, 256, false, false> ScoresB96;
typedef CfgDma<DmaKC<1, 64>, DmaKC<1, 64>, 1, 1, 64, 64, 256, false, false> ScoresB64;
typedef Cfg<LoadKC<3, 128, 1>, LoadKC<3, 128, 1>, 3, 128, 1, 1, 0> ScoresF128;
typedef Cfg<LoadKC<3, 64, 3>, LoadKC<3, 64, 3>, 3, 64, 3, 2, 1> ScoresF64;
typedef CfgMix<DmaKC<2, 128>, LoadKC<2, 128, 1, 256, true>, 128, 128, 256, 2> ScoresH128;
typedef CfgMix<DmaKC<2, 256, 512>, LoadKC<2, 128, 1, 512, true>, 256, 128, 512, 2> ScoresH256;
// dq = g cand, dc = g^T q
typedef CfgDma<DmaKC<2, 128>, DmaKS<1, 128>, 2, 1, 128, 128, 256, false, true> GradQB128;
typedef CfgDma<DmaKS<2, 128>, DmaKS<1, 128>, 2, 1, 128, 128, 256, false, true> GradPB128;
typedef CfgDma<DmaKC<2, 64>, DmaKS<1, 64>, 2, 1, 64, 64, 256, false, true> GradQB64;
typedef CfgDma<DmaKS<2, 64>, DmaKS<1, 64>, 2, 1, 64, 64, 256, false, true> GradPB64;
typedef Cfg<LoadKC<3, 128, 1>, LoadKS<3, 128, 1>, 3, 128, 1, 1, 0> GradQF128;
typedef Cfg<LoadKS<3, 128, 1>, LoadKS<3, 128, 1>, 3, 128, 1, 1, 0> GradPF128;
typedef Cfg<LoadKC<3, 64, 2>, LoadKS<3, 64, 2>, 3, 64, 2, 1, 0> GradQF64;
typedef Cfg<LoadKS<3, 64, 2>, LoadKS<3, 64, 2>, 3, 64, 2, 1, 0> GradPF64;
typedef CfgMix<DmaKC<2, 128>, LoadKS<2, 128, 1>, 128, 128, 256, 1> GradQH128;
typedef CfgDma<DmaKS<2, 128>, DmaKS<2, 128>, 2, 2, 128, 128, 256, true, false> GradPH128;
typedef CfgMix<DmaKC<2, 256, 512>, LoadKS<2, 128, 1, 512>, 256, 128, 512, 0> GradQH256;
typedef CfgDma<DmaKS<2, 256, 512>, DmaKS<2, 128, 512>, 2, 2, 256, 128, 512, true, false> GradPH256;

// 256 rows of a side in one tile, by eight waves, instead of two tiles of 128: fp32 values of the other side are read and split half
// as often (256 x 32768 x 4096, with the kernels around them: scores 221 us for 249, gradients 294 for 311).  Taken where at most a fifth more rows are computed for it.
static GemmArgs tall(GemmArgs g) {
    g.nm = (int)tiles_of(g.a.rows, 256);
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
    unsigned* cnt = (unsigned*)(w + L.off_cnt);
    unsigned* flag = (unsigned*)(w + L.off_flag);
    const int nc = (int)(B + 1 + (B + 31) / 32);
    const Side sq{q, q, B, d, B, d}, sc{p, memory, C, d, T, d};
    GemmArgs g = gemm_args(sq, sc, d, L.s, w, L.lds, B * L.lds);
    const bool ready = L.s.splits == 1;
    if (ready) { g.seg = (float*)(w + L.off_seg); g.segs = L.segs; g.f2 = temp; }
    if (dtype == ABC_DT_BF16) {
        if (L.narrow) launch_scores<ScoresB96>(g, nullptr, 0, nullptr, nullptr, 0, cnt, nc, st);
        else if (L.s.tile == 128) launch_scores<ScoresB128>(g, nullptr, 0, nullptr, nullptr, 0, cnt, nc, st);
        else launch_scores<ScoresB64>(g, nullptr, 0, nullptr, nullptr, 0, cnt, nc, st);
    } else if (L.fast) {
        unsigned* qout = (unsigned*)(w + L.off_qout);
        hipLaunchKernelGGL(distill_split_kernel, dim3((unsigned)B), dim3(256), 0, st, (const float*)q, d, (d + 31) / 32 * 32, teacher_idx, teacher_score, k,
                           w + L.off_q, qout, flag);
        GemmArgs h = g;
        h.a = Side{w + L.off_q, w + L.off_q, B, (d + 31) / 32 * 64, B, (d + 31) / 32 * 32};
        if (tiles_of(B, 256) * 2 * 5 <= tiles_of(B, 128) * 6) launch_scores<ScoresH256>(tall(h), nullptr, 0, flag, qout, B, cnt, nc, st);
        else launch_scores<ScoresH128>(h, nullptr, 0, flag, qout, B, cnt, nc, st);
        launch_scores<ScoresF128>(g, flag, 1, nullptr, nullptr, 0, nullptr, 0, st);
    } else if (L.s.tile == 128) launch_scores<ScoresF128>(g, nullptr, 0, nullptr, nullptr, 0, cnt, nc, st);
    else launch_scores<ScoresF64>(g, nullptr, 0, nullptr, nullptr, 0, cnt, nc, st);
    RowArgs r;
    r.part = (const float*)w; r.s = (float*)(w + L.off_s); r.splits = L.s.splits; r.segs = L.segs; r.ready = ready; r.slab = B * L.lds; r.lds = L.lds;
    r.temp = temp; r.idx = teacher_idx; r.score = teacher_score; r.teacher_temp = teacher_temp; r.B = B; r.T = T; r.k = k;
    r.seg = (float*)(w + L.off_seg); r.norm = (float*)(w + L.off_norm); r.t = (float*)(w + L.off_t); r.li = (int*)(w + L.off_li);
    r.row = (float*)(w + L.off_row); r.stat = (float*)(w + L.off_stat); r.cnt = cnt; r.out_loss = out_loss; r.out_agree = out_agree;
    hipLaunchKernelGGL(distill_row_kernel, dim3(ready ? 1u : (unsigned)L.segs, (unsigned)B), dim3(256), 0, st, r);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ABC_OK : abc_fail_hip(e, "distill_fwd launch");
}

extern "C" int abc_distill_bwd(int dtype, const void* q, const void* p, const void* memory, const float* temp, const float* grad_out,
                               int64_t B, int64_t C, int64_t M, int d, int k, void* dq, void* dp, float* d_temp, const void* fwd_ws,
                               size_t fwd_ws_bytes, void* ws, size_t ws_bytes, void* stream) {
    int rc = distill_check(dtype, B, C, M, d, k);
    if (rc) return rc;
    if (!q || !p || (M && !memory) || !temp || !grad_out || !fwd_ws) return abc_fail_invalid("distill_bwd: null pointer");
    if (((uintptr_t)q | (uintptr_t)p | (uintptr_t)(M ? memory : nullptr) | (uintptr_t)dq | (uintptr_t)dp) & 15)
        return abc_fail_invalid("distill_bwd: embeddings and gradients must be 16-byte aligned");
    const int64_t T = C + M;
    const FwdLayout F = fwd_layout(dtype, B, T, d, k);
    if (fwd_ws_bytes < F.total) return abc_fail_ws(F.total, fwd_ws_bytes);
    const BwdLayout L = bwd_layout(dtype, B, C, T, d, F.fast, dq, dp);
    if (!ws || ws_bytes < L.total) return abc_fail_ws(L.total, ws_bytes);
    if (((uintptr_t)ws | (uintptr_t)fwd_ws) & 15) return abc_fail_invalid("distill_bwd: workspaces must be 16-byte aligned");
    if (!dq && !dp && !d_temp) return ABC_OK;
    hipStream_t st = (hipStream_t)stream;
    const char* f = (const char*)fwd_ws;
    char* w = (char*)ws;
    const bool bf = dtype == ABC_DT_BF16;
    const unsigned* flag = F.fast ? (const unsigned*)(f + F.off_flag) : nullptr;
    const float* stat = (const float*)(f + F.off_stat);
    GradArgs a;
    a.s = (const float*)(f + F.off_s); a.lds = F.lds; a.norm = (const float*)(f + F.off_norm); a.t = (const float*)(f + F.off_t);
    a.li = (const int*)(f + F.off_li); a.has = (const float*)(f + F.off_row) + 2 * B; a.temp = temp;
    a.T = T; a.ldg = L.ldg; a.k = k; a.form = bf ? G_BF16 : F.fast ? G_F16 : G_F32; a.flag = flag;
    a.g = w + L.off_g; a.segs = L.segs; a.dt = (float*)(w + L.off_dt);
    a.q = (const char*)q; a.qlive = w + L.off_ql; a.qbytes = d * (bf ? 2 : 4);
    const int all = L.segs + (dp ? 1 : 0), most = (int)(((1 << 24) - 1) / B);   // a launch has fewer than 2^32 threads
    for (a.seg0 = 0; a.seg0 < all; a.seg0 += most)
        hipLaunchKernelGGL(distill_grad_kernel, dim3((unsigned)min(most, all - a.seg0), (unsigned)B), dim3(256), 0, st, a);
    SumArgs sa = {};
    if (dq || dp) {
        const Side gq{a.g, a.g, B, L.ldg, B, L.ldg}, gp{a.g, a.g, B, L.ldg, C, L.ldg};                       // fp32
        const Side hq{a.g, a.g, B, L.ldg * 2, B, L.ldg}, hp{a.g, a.g, B, L.ldg * 2, C, L.ldg};               // two parts
        const Side cand{p, memory, C, d, d, d}, query{a.qlive, a.qlive, B, d, d, d};
        GemmArgs xq = gemm_args(gq, cand, T, L.q, L.q.splits > 1 ? (void*)(w + L.off_pq) : dq, d, B * d);
        GemmArgs xp = gemm_args(gp, query, B, L.p, L.p.splits > 1 ? (void*)(w + L.off_pp) : dp, d, C * d);
        for (GemmArgs* x : {&xq, &xp}) { x->f0 = grad_out; x->f1 = stat; x->f2 = temp; }
        if (L.q.splits == 1) xq.live = a.has;
        if (bf) {
            xq.a = hq;
            xp.a = hp;
            if (L.q.tile == 128) launch_grads<GradQB128, GradPB128>(xq, xp, dq, dp, nullptr, 0, st);
            else launch_grads<GradQB64, GradPB64>(xq, xp, dq, dp, nullptr, 0, st);
        } else if (F.fast) {
            GemmArgs yq = xq, yp = xp;
            yq.scale = yp.scale = 1.0f / G_SCALE;
            yq.a = hq;
            yp.a = hp;
            yp.b = Side{f + F.off_q, f + F.off_q, B, (d + 31) / 32 * 64, d, (d + 31) / 32 * 32};
            const int64_t wide = (dq ? tiles_of(B, 256) * T : 0) + (dp ? tiles_of(C, 256) * B : 0);
            const int64_t narrow = (dq ? tiles_of(B, 128) * T : 0) + (dp ? tiles_of(C, 128) * B : 0);
            if (wide * 2 * 5 <= narrow * 6) launch_grads<GradQH256, GradPH256>(tall(yq), tall(yp), dq, dp, flag, 0, st);
            else launch_grads<GradQH128, GradPH128>(yq, yp, dq, dp, flag, 0, st);
            launch_grads<GradQF128, GradPF128>(xq, xp, dq, dp, flag, 1, st);
        } else if (L.q.tile == 128) launch_grads<GradQF128, GradPF128>(xq, xp, dq, dp, nullptr, 0, st);
        else launch_grads<GradQF64, GradPF64>(xq, xp, dq, dp, nullptr, 0, st);
        if (dq && L.q.splits > 1) { sa.part[0] = (const float*)(w + L.off_pq); sa.out[0] = dq; sa.n[0] = B * d; sa.splits[0] = L.q.splits; }
        if (dp && L.p.splits > 1) { sa.part[1] = (const float*)(w + L.off_pp); sa.out[1] = dp; sa.n[1] = C * d; sa.splits[1] = L.p.splits; }
    }
    if (sa.n[0] || sa.n[1] || d_temp) {
        sa.blocks0 = (int)((sa.n[0] + 1023) / 1024);
        const int blocks1 = (int)((sa.n[1] + 1023) / 1024);
        sa.dt = a.dt; sa.ndt = B * L.segs; sa.f0 = grad_out; sa.f1 = stat; sa.f2 = temp; sa.d_temp = d_temp; sa.live = a.has; sa.d = d;
        if (bf) hipLaunchKernelGGL(distill_sum_kernel<true>, dim3(sa.blocks0 + blocks1 + 1), dim3(256), 0, st, sa);
        else hipLaunchKernelGGL(distill_sum_kernel<false>, dim3(sa.blocks0 + blocks1 + 1), dim3(256), 0, st, sa);
    }
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ABC_OK : abc_fail_hip(e, "distill_bwd launch");
}
