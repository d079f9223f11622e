// A store of embeddings held in 4 or 8 bits, for gfx950 (MI355X): rows are quantised as they are written into slots, rows are
// read back by index, and a few queries are scored against every row of the 4-bit form.
//
//   i8    scale = max|x| / 127 (1 where that is zero), code = clamp(rint(x / scale), -127, 127): abc_quantize_i8's rule, so the
//         search kernels contract the rows as they lie.
//   fp4   groups of g = 32 / 64 / 128 values; scale = max(bf16(max|x| / 6), 2^-120); a value is held as the nearest of
//         {0, .5, 1, 1.5, 2, 3, 4, 6} * scale (e2m1 codes 0..7, ties to the even code, sign in bit 3).  The scale carries 8
//         significant bits and a midpoint between two levels at most 3, so every midpoint * scale is exact in fp32 and the
//         comparisons below find the nearest level of the exact quotient.  (Rounding the scale down leaves max|x| / scale a little
//         over 6: the largest code.)  The floor 2^-120 keeps the midpoints out of the subnormal range.
//   A row or group that holds an infinity or a NaN gets a NaN scale: what is read back or scored from it is NaN.
//
// fp4 layout: a row is padded with zeros to pieces of 128 values = 64 bytes.  Value k = 32 m + 8 c + j (m, c < 4, j < 8) of a piece
// is nibble 32 c + 8 m + j, low nibble first: a lane of the scoring kernel (row = lane % 16, c = lane / 16) loads 16 bytes and holds,
// in word m, exactly the 8 values of its B fragment for the m-th 16x16x32 MFMA, whose 32 values lie in one scale group.
#include "common.h"
#include "../../include/abcsearch.h"
#include <type_traits>

int abc_fail_hip(hipError_t e, const char* where);
int abc_fail_invalid(const char* msg);
int abc_fail_ws(size_t need, size_t have);

#define STORE_MAX_DIM 8192
#define SCORE_LDS 163840              // a workgroup's LDS in the scoring kernel: a CU's
// writes of up to this many rows look for repeated slots inside the writing kernel (fp4/128, us, with the claims' two launches: 1024 x 4096 6.4 /
// 9.7, 2048 x 4096 10.8 / 13.7, 4096 x 4096 22 / 21)
#define STORE_SCAN_MAX 2048

typedef __attribute__((ext_vector_type(8))) __bf16 v8bf;
typedef __attribute__((ext_vector_type(2))) __bf16 v2bf;
typedef __attribute__((ext_vector_type(4))) unsigned int v4u;
typedef __attribute__((ext_vector_type(2))) unsigned int v2u;
// rows of any width start at any multiple of the element: the hardware takes wide accesses at such addresses
typedef v4f v4f_u __attribute__((aligned(4)));
typedef v4u v4u_u __attribute__((aligned(2)));

// values k .. k+7 of a row, zeros past its end
template <bool BF16>
__device__ __forceinline__ void load8(const void* row, int k, int dim, float (&v)[8]) {
    if (k + 8 <= dim) {
        if constexpr (BF16) {
            const v4u w = *(const v4u_u*)((const uint16_t*)row + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u); }
        } else {
            const v4f a = *(const v4f_u*)((const float*)row + k), b = *(const v4f_u*)((const float*)row + k + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (BF16) v[j] = k + j < dim ? __uint_as_float((uint32_t)((const uint16_t*)row)[k + j] << 16) : 0.f;
            else v[j] = k + j < dim ? ((const float*)row)[k + j] : 0.f;
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void store8(void* row, int k, int dim, const float (&v)[8]) {
    if (k + 8 <= dim) {
        if constexpr (BF16) {
            v4u w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16_bits(v[2 * j]) | (f32_to_bf16_bits(v[2 * j + 1]) << 16);
            *(v4u_u*)((uint16_t*)row + k) = w;
        } else {
            *(v4f_u*)((float*)row + k) = v4f{v[0], v[1], v[2], v[3]};
            *(v4f_u*)((float*)row + k + 4) = v4f{v[4], v[5], v[6], v[7]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < dim) {
                if constexpr (BF16) ((uint16_t*)row)[k + j] = (uint16_t)f32_to_bf16_bits(v[j]);
                else ((float*)row)[k + j] = v[j];
            }
    }
}

// ---- writing -----------------------------------------------------------------------------------------------------------
struct StoreWriteArgs {
    const void* x;
    int64_t ldx;                    // elements
    const int64_t* slots;           // null: slot i = (first + i) % capacity
    int64_t first, n, capacity;
    int dim, width;                 // width: dim rounded up to 128
    void* data;
    void* scale;
    const int32_t* claim;           // claim[slot] = the last row that names it (null: the kernel looks through `slots` itself)
    int tx;                         // threads a row (a power of two, 16..256)
    int64_t row0;                   // first row of this launch
};

// Rows that name the same slot: the last one is the one that stays, as when the rows are written one after another.
__global__ void store_claim_clear_kernel(const int64_t* __restrict__ slots, int64_t n, int64_t capacity, int32_t* __restrict__ claim) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n && slots[i] >= 0 && slots[i] < capacity) claim[slots[i]] = -1;
}
__global__ void store_claim_kernel(const int64_t* __restrict__ slots, int64_t n, int64_t capacity, int32_t* __restrict__ claim) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n && slots[i] >= 0 && slots[i] < capacity) atomicMax(claim + slots[i], (int32_t)i);
}

// nearest level of |x| / s as a code 0..7 (see the head of the file)
__device__ __forceinline__ uint32_t fp4_code(float a, float s) {
    return (uint32_t)(a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) + (a >= 1.75f * s) + (a > 2.5f * s) + (a >= 3.5f * s) + (a > 5.0f * s);
}

// GROUP 0: i8; otherwise fp4 groups of GROUP values.  A row belongs to tx threads, each of which holds 8 neighbouring values at a
// time; a workgroup of 256 threads takes 256 / tx rows.  i8 needs the whole row before the first code: up to 4 pieces of 8 a thread
// stay in registers (8192 values / 256 threads).
template <bool BF16, int GROUP>
__global__ __launch_bounds__(256) void store_write_kernel(const StoreWriteArgs a) {
    __shared__ uint32_t red[4];
    const int tx = a.tx, t = threadIdx.x & (tx - 1);
    const int64_t row = a.row0 + (int64_t)blockIdx.x * (256 / tx) + threadIdx.x / tx;
    const bool live = row < a.n;
    int64_t slot = -1;
    if (live) slot = a.slots ? a.slots[row] : (a.first + row) % a.capacity;
    bool on = live && slot >= 0 && slot < a.capacity;
    if (a.slots && a.n > 1) {
        if (a.claim) {
            on = on && a.claim[slot] == (int32_t)row;
        } else {
            bool again = false;                                  // a later row names this slot
            if (on)
                for (int64_t j = row + 1 + t; j < a.n; j += tx) again |= a.slots[j] == slot;
            if (tx <= 64) {
                for (int m = 1; m < tx; m <<= 1) again |= (bool)__shfl_xor((int)again, m, 64);
                on = on && !again;
            } else {
                // a workgroup of more than one wave a row: 256 / tx rows share the barrier, each with its waves' flags
                const int wave = threadIdx.x >> 6;
                const bool any = __any(again);
                if ((threadIdx.x & 63) == 0) red[wave] = any;
                __syncthreads();
                const int w0 = (threadIdx.x / tx) * (tx / 64);
                for (int w = 0; w < tx / 64; ++w) on = on && !red[w0 + w];
                __syncthreads();
            }
        }
    }
    const char* xr = (const char*)a.x + (live ? row : 0) * a.ldx * (BF16 ? 2 : 4);
    const int pieces = a.width / 8;
    if constexpr (GROUP > 0) {
        uint32_t* out = (uint32_t*)((char*)a.data + (on ? slot : 0) * (int64_t)(a.width / 2));
        uint16_t* os = (uint16_t*)a.scale + (on ? slot : 0) * (int64_t)(a.width / GROUP);
        for (int p = t; p < pieces; p += tx) {                   // pieces is a multiple of 16: a group's lanes stay together
            float v[8];
            load8<BF16>(xr, p * 8, live ? a.dim : 0, v);
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);   // infinities and NaN are the largest
#pragma unroll
            for (int m = 1; m < GROUP / 8; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
            uint32_t word = 0, sbits = 0x7FC0u;
            if (top < 0x7F800000u) {
                sbits = f32_to_bf16_bits(__fdiv_rn(__uint_as_float(top), 6.0f));
                float s = __uint_as_float(sbits << 16);
                if (s < 0x1p-120f) { s = 0x1p-120f; sbits = 0x0380u; }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    word |= (fp4_code(fabsf(v[j]), s) | (v[j] < 0.f ? 8u : 0u)) << (4 * j);
            }
            if (on) {
                out[(p >> 4) * 16 + (p & 3) * 4 + ((p >> 2) & 3)] = word;
                if ((p & (GROUP / 8 - 1)) == 0) os[p / (GROUP / 8)] = (uint16_t)sbits;
            }
        }
    } else {
        float v[4][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            load8<BF16>(xr, (t + i * tx) * 8, live ? a.dim : 0, v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
        }
        for (int m = 1; m < (tx < 64 ? tx : 64); m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
        if (tx > 64) {
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
            __syncthreads();
            const int w0 = (threadIdx.x / tx) * (tx / 64);
            for (int w = 0; w < tx / 64; ++w) top = max(top, red[w0 + w]);
        }
        if (!on) return;
        const bool bad = top >= 0x7F800000u;
        float s = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(__uint_as_float(top), 127.0f);
        if (s == 0.f) s = 1.0f;                                  // a row of zeros, or one whose largest value is below 2^-143
        char* out = (char*)a.data + slot * (int64_t)a.width;
        if (t == 0) ((float*)a.scale)[slot] = s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t + i * tx;
            if (p >= pieces) continue;
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float r = bad ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(v[i][j], s)), -127.f), 127.f);
                w[j >> 2] |= (uint32_t)(uint8_t)(int8_t)r << (8 * (j & 3));
            }
            *(v2u*)(out + p * 8) = v2u{w[0], w[1]};
        }
    }
}

static int store_check(int64_t capacity, int dim, int group) {
    if (capacity < 0 || capacity > 0x7FFFFFFFll) return abc_fail_invalid("store: capacity out of range [0, 2^31)");
    if (dim < 1 || dim > STORE_MAX_DIM) return abc_fail_invalid("store: dim out of range [1, 8192]");
    if (group != 0 && group != 32 && group != 64 && group != 128) return abc_fail_invalid("store: group must be 32, 64 or 128 (0 = the 8-bit form)");
    return ABC_OK;
}

static int row_threads(int pieces) {
    int tx = 16;
    while (tx < 256 && tx < pieces) tx <<= 1;
    return tx;
}

// A launch has fewer than 2^32 threads: rows a launch, and its workgroups for n rows from row0 on.
static int64_t rows_a_launch(int tx) { return (int64_t)(1 << 23) * (256 / tx); }
static unsigned row_groups(int64_t n, int64_t row0, int tx) {
    const int64_t m = n - row0 < rows_a_launch(tx) ? n - row0 : rows_a_launch(tx);
    return (unsigned)((m + 256 / tx - 1) / (256 / tx));
}

extern "C" size_t abc_store_write_workspace_bytes(int64_t n, int64_t capacity) {
    if (n <= STORE_SCAN_MAX || capacity <= 0) return 0;
    return (size_t)capacity * 4;
}

extern "C" int abc_store_write(int x_dtype, const void* x, int64_t ldx, const int64_t* slots, int64_t first, int64_t n, int dim,
                               void* data, void* scale, int64_t capacity, int group, void* ws, size_t ws_bytes, void* stream) {
    int rc = store_check(capacity, dim, group);
    if (rc) return rc;
    if (x_dtype != ABC_DT_F32 && x_dtype != ABC_DT_BF16) return abc_fail_invalid("store_write: rows must be f32 or bf16");
    if (n < 0 || n > 0x7FFFFFFFll) return abc_fail_invalid("store_write: row count out of range [0, 2^31)");
    if (n == 0) return ABC_OK;
    if (!x || !data || !scale) return abc_fail_invalid("store_write: null pointer");
    if (ldx < dim) return abc_fail_invalid("store_write: row stride below dim");
    if ((uintptr_t)data & 15) return abc_fail_invalid("store_write: data must be 16-byte aligned");
    if ((uintptr_t)scale & (group ? 1 : 3)) return abc_fail_invalid("store_write: scale must be aligned to its element");
    if (!slots && (first < 0 || first >= capacity || n > capacity)) return abc_fail_invalid("store_write: run of slots out of range");
    const size_t need = slots ? abc_store_write_workspace_bytes(n, capacity) : 0;
    if (need && (!ws || ws_bytes < need)) return abc_fail_ws(need, ws_bytes);
    hipStream_t st = (hipStream_t)stream;
    StoreWriteArgs a;
    a.x = x; a.ldx = ldx; a.slots = slots; a.first = first; a.n = n; a.capacity = capacity;
    a.dim = dim; a.width = (dim + 127) / 128 * 128;
    a.data = data; a.scale = scale; a.claim = need ? (const int32_t*)ws : nullptr;
    a.tx = row_threads(a.width / 8);
    if (need) {
        const unsigned g = (unsigned)((n + 255) / 256);
        hipLaunchKernelGGL(store_claim_clear_kernel, dim3(g), dim3(256), 0, st, slots, n, capacity, (int32_t*)ws);
        hipLaunchKernelGGL(store_claim_kernel, dim3(g), dim3(256), 0, st, slots, n, capacity, (int32_t*)ws);
    }
    const bool bf = x_dtype == ABC_DT_BF16;
#define STORE_WRITE(G) do { if (bf) hipLaunchKernelGGL((store_write_kernel<true, G>), dim3(grid), dim3(256), 0, st, a); \
                            else hipLaunchKernelGGL((store_write_kernel<false, G>), dim3(grid), dim3(256), 0, st, a); } while (0)
    for (a.row0 = 0; a.row0 < n; a.row0 += rows_a_launch(a.tx)) {
        const unsigned grid = row_groups(n, a.row0, a.tx);
        if (group == 0) STORE_WRITE(0);
        else if (group == 32) STORE_WRITE(32);
        else if (group == 64) STORE_WRITE(64);
        else STORE_WRITE(128);
    }
#undef STORE_WRITE
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ABC_OK : abc_fail_hip(e, "store_write launch");
}

// ---- reading -----------------------------------------------------------------------------------------------------------
struct StoreReadArgs {
    const int64_t* index;           // null: row i = first + i
    int64_t first, n, capacity;
    const void* data;
    const void* scale;
    int dim, width, tx;
    void* out;
    int64_t ldo;
    int64_t row0;                   // first row of this launch
};

// the 8 fp32 values of one word of e2m1 codes, times s (exact: 2 significant bits times 8)
__device__ __forceinline__ void fp4_values(uint32_t w, float s, float (&v)[8]) {
#define FP4_PAIR(b) do { const v2bf p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, b); v[2 * b] = (float)p[0] * s; v[2 * b + 1] = (float)p[1] * s; } while (0)
    FP4_PAIR(0); FP4_PAIR(1); FP4_PAIR(2); FP4_PAIR(3);
#undef FP4_PAIR
}

// HBM-bound: held bytes in, dim * sizeof(out) bytes out.  Index < 0: a row of zeros; index >= capacity: a row of NaN.
template <bool BF16, int GROUP>
__global__ __launch_bounds__(256) void store_read_kernel(const StoreReadArgs a) {
    const int tx = a.tx, t = threadIdx.x & (tx - 1);
    const int64_t i = a.row0 + (int64_t)blockIdx.x * (256 / tx) + threadIdx.x / tx;
    if (i >= a.n) return;
    const int64_t row = a.index ? a.index[i] : a.first + i;
    char* out = (char*)a.out + i * a.ldo * (BF16 ? 2 : 4);
    const int pieces = (a.dim + 7) / 8;
    if (row < 0 || row >= a.capacity) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = row < 0 ? 0.f : __uint_as_float(0x7FC00000u);
        for (int p = t; p < pieces; p += tx) store8<BF16>(out, p * 8, a.dim, v);
        return;
    }
    if constexpr (GROUP > 0) {
        const uint32_t* src = (const uint32_t*)((const char*)a.data + row * (int64_t)(a.width / 2));
        const uint16_t* sc = (const uint16_t*)a.scale + row * (int64_t)(a.width / GROUP);
        for (int p = t; p < pieces; p += tx) {
            float v[8];
            fp4_values(src[(p >> 4) * 16 + (p & 3) * 4 + ((p >> 2) & 3)], __uint_as_float((uint32_t)sc[p / (GROUP / 8)] << 16), v);
            store8<BF16>(out, p * 8, a.dim, v);
        }
    } else {
        const char* src = (const char*)a.data + row * (int64_t)a.width;
        const float s = ((const float*)a.scale)[row];
        for (int p = 2 * t; p < pieces; p += 2 * tx) {           // 16 codes a lane
            const v4u w = *(const v4u*)(src + p * 8);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (float)(int8_t)(w[2 * h + (j >> 2)] >> (8 * (j & 3))) * s;
                store8<BF16>(out, (p + h) * 8, a.dim, v);
            }
        }
    }
}

extern "C" int abc_store_read(const int64_t* index, int64_t first, int64_t n, const void* data, const void* scale, int64_t capacity,
                              int dim, int group, int out_dtype, void* out, int64_t ldo, void* stream) {
    int rc = store_check(capacity, dim, group);
    if (rc) return rc;
    if (out_dtype != ABC_DT_F32 && out_dtype != ABC_DT_BF16) return abc_fail_invalid("store_read: rows are read as f32 or bf16");
    if (n < 0 || n > 0x7FFFFFFFll) return abc_fail_invalid("store_read: row count out of range [0, 2^31)");
    if (n == 0) return ABC_OK;
    if (!out || (capacity > 0 && (!data || !scale))) return abc_fail_invalid("store_read: null pointer");
    if (ldo < dim) return abc_fail_invalid("store_read: row stride below dim");
    if ((uintptr_t)data & 15) return abc_fail_invalid("store_read: data must be 16-byte aligned");
    if (!index && (first < 0 || first + n > capacity)) return abc_fail_invalid("store_read: run of rows out of range");
    StoreReadArgs a;
    a.index = index; a.first = first; a.n = n; a.capacity = capacity; a.data = data; a.scale = scale;
    a.dim = dim; a.width = (dim + 127) / 128 * 128; a.out = out; a.ldo = ldo;
    a.tx = row_threads(group ? (dim + 7) / 8 : (dim + 15) / 16);
    hipStream_t st = (hipStream_t)stream;
    const bool bf = out_dtype == ABC_DT_BF16;
#define STORE_READ(G) do { if (bf) hipLaunchKernelGGL((store_read_kernel<true, G>), dim3(grid), dim3(256), 0, st, a); \
                           else hipLaunchKernelGGL((store_read_kernel<false, G>), dim3(grid), dim3(256), 0, st, a); } while (0)
    for (a.row0 = 0; a.row0 < n; a.row0 += rows_a_launch(a.tx)) {
        const unsigned grid = row_groups(n, a.row0, a.tx);
        if (group == 0) STORE_READ(0);
        else if (group == 32) STORE_READ(32);
        else if (group == 64) STORE_READ(64);
        else STORE_READ(128);
    }
#undef STORE_READ
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ABC_OK : abc_fail_hip(e, "store_read launch");
}

// ---- scores of a few queries against the fp4 form ------------------------------------------------------------------------
struct StoreScoreArgs {
    const void* q;
    int64_t ldq;
    int nq;                         // queries of this launch
    const char* data;
    const uint16_t* scale;
    int64_t rows;
    int dim, chunks;                // chunks: pieces of 128 values a row
    int slice;                      // chunks of the queries that LDS holds at a time
    int ks;                         // waves that share a tile of 16 rows, each with its share of the chunks
    float* out;
    int64_t ldo;
};

// fp32 = hi + mid + lo, three bf16 values that carry its 24 significant bits: hi is cut (never past the largest bf16), the rest
// rounded.  What an infinity or a NaN leaves in mid and lo is set to zero, so that the products with hi alone carry it on.
__device__ __forceinline__ void split3(float x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    const uint32_t u = __float_as_uint(x);
    const bool fin = (u & 0x7F800000u) != 0x7F800000u;
    hi = u >> 16;
    if (!fin && (u & 0x007FFFFFu)) hi |= 0x40u;
    const float r = fin ? x - __uint_as_float(u & 0xFFFF0000u) : 0.f;
    mid = f32_to_bf16_bits(r);
    lo = f32_to_bf16_bits(r - __uint_as_float(mid << 16));
}

// Memory-bound with few queries: dim / 2 bytes of codes and 256 / GROUP bytes of scales a 128 values stream through once, whatever the
// number of queries up to 16 fp32 (64 bf16).  A wave owns a tile of 16 rows: its lanes load 16 bytes of codes, four conversions a word
// make a bf16 B fragment of them (e2m1 values are exact in bf16), and 16x16x32 MFMAs multiply it with the queries' fragments out of LDS.
// fp32 queries stand in LDS as three bf16 parts (24 bits).  Up to four: in rows 4 q + part of one A tile, so that a lane's accumulators
// hold the parts' sums of one query.  Up to sixteen: a part an A tile, all three into one accumulator, the smallest part first (13
// queries, 100 003 x 1000: 21 us; four queries a tile, four tiles, reads a third more LDS and spills: 30 us).  Products and sums are
// fp32.  A group's sum is scaled once.  The loads of the next four pieces (the next tile's, at a tile's end) are on their way while
// four are multiplied: 4 KB a wave, 64 KB a CU.  Scales come 16 bytes a lane, 32 of a row at a time, and go through a strip of LDS
// of the wave's own (read where they are needed, 2 bytes a lane, they cost a third of the time: every access touches 16 lines).
// 1 x 412 500 x 4096: 149 us, 5.8 TB/s.  More queries than LDS holds whole (fp32: more than 4 of 4096 values, 16 of 1000; bf16: more than 16 of
// 4096) go in slices of the row: for every round of tiles each slice is read, split and put into LDS again between two barriers, and the
// loads of codes do not go on across them.  That is the step in 103 000 x 4096, 1 / 4 / 6 / 13 fp32 queries 36 / 39 / 61 / 76 us, 16 / 32 / 64 bf16 42 / 63 /
// 121 us (412 500 rows: 150 / 165 / 246 / 304 and 186 / 266 / 441).
#define SCORE_WAVES 16               // a workgroup: all that a CU holds of this kernel, so that the queries stand in its LDS once
#define SCORE_STRIP 1280             // bytes of scales a wave: 16 rows of 32, 80 bytes apart
// between a query part's rows in LDS.  64, with the four 16-byte chunks of a fragment's 64 bytes permuted with the row: a fragment's 16 lanes
// of a phase ({0-3, 12-15, 20-27}, {4-11, 16-19, 28-31}) touch all banks once
#define SCORE_PAD(full) ((full) ? 64 : 16)

template <int GROUP>
struct ScorePieces {
    static constexpr int G = 128 / GROUP;
    v4u code[4];
    // four pieces of a row from piece cb on, n of them there (scalar, at least 1): the last again past them
    __device__ __forceinline__ void fetch(const char* dr, int cb, int n) {
#pragma unroll
        for (int u = 0; u < 4; ++u) code[u] = *(const v4u*)(dr + (cb + (u < n ? u : n - 1)) * 64);
    }
};
// 8 of the 32 scales from `at` on (in 2-byte units from the first row's first scale; `total` of them in all)
__device__ __forceinline__ v4u fetch_scales(const uint16_t* scale, int64_t at, int64_t total) {
    if (at + 8 <= total) return *(const v4u_u*)(scale + at);
    v4u w = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (at + j < total) w[j >> 1] |= (uint32_t)scale[at + j] << (16 * (j & 1));
    return w;
}

template <bool QBF16, int GROUP, int MT>
__global__ __launch_bounds__(64 * SCORE_WAVES) void store_scores_kernel(const StoreScoreArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    constexpr bool SIDE = !QBF16 && MT == 3;                     // the parts of 16 fp32 queries in A tiles of their own, one accumulator
    constexpr bool FULL = QBF16 || SIDE;                         // a lane's accumulators hold four queries' scores
    constexpr int P = QBF16 ? 1 : 3, G = 128 / GROUP, R = FULL ? 4 : 3, NT = SIDE ? 1 : MT;   // R: accumulators of a lane that mean something
    constexpr int EACH = 8 / G;                                  // groups of four pieces that 32 scales of a row serve
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l15 = lane & 15, c = lane >> 4;
    char* strip = smem_raw + wave * SCORE_STRIP;
    char* const qlds = smem_raw + SCORE_WAVES * SCORE_STRIP;
    const int pitch = a.slice * 256 + SCORE_PAD(FULL);           // bytes a query part
    const int nq4 = (a.nq + 3) & ~3, lrows = SIDE ? 3 * nq4 : a.nq * P;
    typedef typename std::conditional<FULL, v4f, float>::type red_t;       // parts in one tile: they are summed first
    red_t* red = (red_t*)(qlds + lrows * pitch);
    const int ks = wave & (a.ks - 1), sub = wave / a.ks, per = SCORE_WAVES / a.ks;
    const int64_t tiles = (a.rows + 15) / 16;
    const int nslices = (a.chunks + a.slice - 1) / a.slice;
    int arow[MT];                                                // byte offset of this lane's row of each A tile
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if constexpr (FULL) {
            const int qi = min(SIDE ? l15 : t * 16 + l15, a.nq - 1);
            arow[t] = ((SIDE ? t * nq4 : 0) + qi) * pitch + ((c ^ (0 - (qi >> 2))) & 3) * 16;
        } else {
            int qi = t * 4 + (l15 >> 2); if (qi >= a.nq) qi = a.nq - 1;
            int part = l15 & 3; if (part > 2) part = 2;
            arow[t] = (qi * 3 + part) * pitch + c * 16;
        }
    }
    auto fill = [&](int s) {
        const int c0 = s * a.slice, nc = min(a.slice, a.chunks - c0);
        for (int i = threadIdx.x; i < a.nq * nc * 16; i += 64 * SCORE_WAVES) {
            const int qi = i / (nc * 16), p = i - qi * (nc * 16);
            float v[8];
            load8<QBF16>((const char*)a.q + qi * a.ldq * (QBF16 ? 2 : 4), (c0 * 16 + p) * 8, a.dim, v);
            char* dst = qlds + (SIDE ? qi : qi * P) * pitch + (FULL ? (p & ~3) | ((p ^ (0 - (qi >> 2))) & 3) : p) * 16;
            const int part = SIDE ? nq4 * pitch : pitch;
            if constexpr (QBF16) {
                v4u w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (__float_as_uint(v[2 * j]) >> 16) | (__float_as_uint(v[2 * j + 1]) & 0xFFFF0000u);
                *(v4u*)dst = w;
            } else {
                uint32_t h[8], m[8], l[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) split3(v[j], h[j], m[j], l[j]);
                *(v4u*)dst = v4u{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
                *(v4u*)(dst + part) = v4u{m[0] | m[1] << 16, m[2] | m[3] << 16, m[4] | m[5] << 16, m[6] | m[7] << 16};
                *(v4u*)(dst + 2 * part) = v4u{l[0] | l[1] << 16, l[2] | l[3] << 16, l[4] | l[5] << 16, l[6] | l[7] << 16};
            }
        }
    };
    auto row_of = [&](int64_t tile) { const int64_t n = tile * 16 + l15; return n < a.rows ? n : a.rows - 1; };
    auto data_of = [&](int64_t row) { return a.data + row * (int64_t)(a.chunks * 64) + c * 16; };
    const int64_t total = a.rows * (int64_t)(a.chunks * G);
    auto scales = [&](int64_t row, int cb) { return fetch_scales(a.scale, (row * a.chunks + cb) * G + c * 8, total); };
    // the waves that share a tile take runs of pieces of a slice
    auto first_of = [&](int c0, int c1, int w) { return c0 + min(c1 - c0, w * ((c1 - c0 + a.ks - 1) / a.ks)); };

    v4f sum[NT];
    ScorePieces<GROUP> cur, next;
    v4u nscale = {0, 0, 0, 0};
    // at: the first piece's place in the queries' LDS; j: the group's place in the strip
    auto multiply = [&](int at, int j, int n) {
        uint32_t sc[2 * G];
        if constexpr (G == 1) { const v2u w = *(const v2u*)(strip + l15 * 80 + j * 8); sc[0] = w[0]; sc[1] = w[1]; }
        else {
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
                const v4u w = *(const v4u*)(strip + l15 * 80 + j * 8 * G + i * 16);
                sc[4 * i] = w[0]; sc[4 * i + 1] = w[1]; sc[4 * i + 2] = w[2]; sc[4 * i + 3] = w[3];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int lbase = at + u * 256;
            if (u >= n) continue;
#pragma unroll
            for (int group = 0; group < G; ++group) {
                union { v8bf f; v2bf h[4]; } b[4 / G];
#pragma unroll
                for (int m = 0; m < 4 / G; ++m) {
                    const uint32_t w = cur.code[u][group * (4 / G) + m];
                    b[m].h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0);
                    b[m].h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1);
                    b[m].h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2);
                    b[m].h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3);
                }
                const int k = u * G + group;
                const float f = __uint_as_float((k & 1) ? (sc[k / 2] & 0xFFFF0000u) : (sc[k / 2] << 16));
                v4f acc;
#pragma unroll
                for (int t = MT - 1; t >= 0; --t) {              // SIDE: the smallest parts first, their sum is rounded at the size it has then
                    if (!SIDE || t == MT - 1) acc = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int m = 0; m < 4 / G; ++m) {
                        const v8bf av = *(const v8bf*)(qlds + arow[t] + lbase + (group * (4 / G) + m) * 64);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, b[m].f, acc, 0, 0, 0);
                    }
                    if (!SIDE || t == 0)
#pragma unroll
                        for (int r = 0; r < R; ++r) sum[SIDE ? 0 : t][r] = fmaf(f, acc[r], sum[SIDE ? 0 : t][r]);
                }
                if (MT > 2 && !SIDE) __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_sched_barrier(0);                   // fragments of one piece at a time: four waves a SIMD hide their reads
        }
    };

    const bool whole = nslices == 1;                             // the queries stand in LDS for good
    const int64_t first0 = blockIdx.x, step = (int64_t)gridDim.x * per;   // neighbouring tiles on different CUs: each gets as many
    if (whole) {
        const int w0 = first_of(0, a.chunks, ks), w1 = first_of(0, a.chunks, ks + 1);
        const int64_t tile = first0 + (int64_t)sub * gridDim.x;
        if (tile < tiles && w0 < w1) {
            const int64_t row = row_of(tile);
            nscale = scales(row, w0);
            next.fetch(data_of(row), w0, w1 - w0);
        }
        fill(0);
        __syncthreads();
    }
    // every workgroup makes the same number of rounds for all of its waves: the barriers inside are met by all of them
    for (int64_t first = first0; first < tiles; first += step) {
        const int64_t tile = first + (int64_t)sub * gridDim.x;
        const int64_t n = tile * 16 + l15;
#pragma unroll
        for (int t = 0; t < NT; ++t) sum[t] = v4f{0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < nslices; ++s) {
            const int c0 = s * a.slice, c1 = min(a.chunks, c0 + a.slice);
            const int e0 = first_of(c0, c1, ks), e1 = first_of(c0, c1, ks + 1);
            const int64_t row = row_of(tile < tiles ? tile : tiles - 1);
            const char* dr = data_of(row);
            if (!whole) {
                if (e0 < e1) {
                    nscale = scales(row, e0);
                    next.fetch(dr, e0, e1 - e0);
                }
                __syncthreads();                                 // the last slice has been read
                fill(s);
                __syncthreads();
            }
            if (tile >= tiles) continue;
            for (int cb = e0, j = 0; cb < e1; cb += 4) {
                cur = next;
                if (j == 0) *(v4u*)(strip + l15 * 80 + c * 16) = nscale;     // (a wave's LDS accesses are carried out in order)
                const int jn = j + 1 == EACH ? 0 : j + 1;
                if (cb + 4 < e1) {
                    if (jn == 0) nscale = scales(row, cb + 4);
                    next.fetch(dr, cb + 4, e1 - cb - 4);
                } else if (whole && tile + step < tiles) {
                    const int64_t r2 = row_of(tile + step);
                    nscale = scales(r2, e0);
                    next.fetch(data_of(r2), e0, e1 - e0);
                }
                multiply((cb - c0) * 256, j, e1 - cb);
                j = jn;
            }
        }
        red_t res[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (FULL) res[t] = sum[t];
            else res[t] = (sum[t][2] + sum[t][1]) + sum[t][0];
        }
        if (a.ks > 1) {                                          // the waves that share the tile, in fixed order
#pragma unroll
            for (int t = 0; t < NT; ++t) red[(wave * NT + t) * 64 + lane] = res[t];
            __syncthreads();
            if (ks == 0) {
                for (int w = 1; w < a.ks; ++w)
#pragma unroll
                    for (int t = 0; t < NT; ++t) res[t] += red[((wave + w) * NT + t) * 64 + lane];
            }
            __syncthreads();
        }
        if (ks == 0 && n < a.rows && tile < tiles) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (FULL) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int qi = t * 16 + 4 * c + r;
                        if (qi < a.nq) a.out[(int64_t)qi * a.ldo + n] = res[t][r];
                    }
                } else {
                    const int qi = t * 4 + c;
                    if (qi < a.nq) a.out[(int64_t)qi * a.ldo + n] = res[t];
                }
            }
        }
    }
}

template <bool QBF16, int GROUP, int MT>
static hipError_t scores_launch_mt(const StoreScoreArgs& a, unsigned grid, size_t lds, hipStream_t st) {
    if (lds > 65536) {                                            // of the current device's copy of the kernel
        const hipError_t e = hipFuncSetAttribute((const void*)store_scores_kernel<QBF16, GROUP, MT>, hipFuncAttributeMaxDynamicSharedMemorySize, SCORE_LDS);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((store_scores_kernel<QBF16, GROUP, MT>), dim3(grid), dim3(64 * SCORE_WAVES), lds, st, a);
    return hipGetLastError();
}
template <bool QBF16, int GROUP>
static hipError_t scores_launch(const StoreScoreArgs& a, int mt, unsigned grid, size_t lds, hipStream_t st) {
    if (mt == 1) return scores_launch_mt<QBF16, GROUP, 1>(a, grid, lds, st);
    if constexpr (QBF16) {
        if (mt == 2) return scores_launch_mt<QBF16, GROUP, 2>(a, grid, lds, st);
        if (mt == 4) return scores_launch_mt<QBF16, GROUP, 4>(a, grid, lds, st);
    }
    return scores_launch_mt<QBF16, GROUP, 3>(a, grid, lds, st);
}

extern "C" int abc_store_scores(int q_dtype, const void* q, int64_t ldq, int64_t nq, const void* data, const void* scale, int64_t rows,
                                int dim, int group, float* out, int64_t ldo, void* stream) {
    int rc = store_check(rows, dim, group);
    if (rc) return rc;
    if (group == 0) return abc_fail_invalid("store_scores: the 4-bit form only (the 8-bit form is searched by abc_topk_i8)");
    if (q_dtype != ABC_DT_F32 && q_dtype != ABC_DT_BF16) return abc_fail_invalid("store_scores: queries must be f32 or bf16");
    if (nq < 0) return abc_fail_invalid("store_scores: negative query count");
    if (nq == 0 || rows == 0) return ABC_OK;
    if (!q || !data || !scale || !out) return abc_fail_invalid("store_scores: null pointer");
    if (ldq < dim || ldo < rows) return abc_fail_invalid("store_scores: row stride below the row's length");
    if (((uintptr_t)data & 15) || ((uintptr_t)scale & (256 / group - 1)))
        return abc_fail_invalid("store_scores: data must be 16-byte aligned, scale to the scales of 128 values");
    hipStream_t st = (hipStream_t)stream;
    const bool bf = q_dtype == ABC_DT_BF16;
    const int chunks = (dim + 127) / 128, most = bf ? 64 : 16;
    const int64_t passes = (nq + most - 1) / most;
    for (int64_t p = 0; p < passes; ++p) {
        const int64_t q0 = nq * p / passes, q1 = nq * (p + 1) / passes;
        StoreScoreArgs a;
        a.nq = (int)(q1 - q0);
        a.q = (const char*)q + q0 * ldq * (bf ? 2 : 4); a.ldq = ldq;
        a.data = (const char*)data; a.scale = (const uint16_t*)scale; a.rows = rows;
        a.dim = dim; a.chunks = chunks; a.out = out + q0 * ldo; a.ldo = ldo;
        const int mt = bf ? (a.nq + 15) / 16 : a.nq <= 4 ? 1 : 3;
        const bool full = bf || mt == 3;
        const int lrows = bf ? a.nq : mt == 3 ? (a.nq + 3) / 4 * 12 : a.nq * 3, nt = bf ? mt : 1;
        // LDS: the waves' strips of scales, the queries (in slices of a row where they are too many), the sums of waves that share a tile
        const int64_t tiles = (rows + 15) / 16;
        int slice = 0, ks = 1;
        size_t red = 0;
        auto fit = [&] {                                          // 1 piece at least: 64 rows of 320 bytes fit beside 84 KB
            slice = (int)((SCORE_LDS - SCORE_WAVES * SCORE_STRIP - red) / lrows - SCORE_PAD(full)) / 256;
            if (slice > chunks) slice = chunks;
        };
        fit();
        // several waves a tile where there are fewer than 2048 (1 x 5000 x 3584: 6.9 us, one wave a tile 16.5; 1 x 30 000: 15.0 and 17.2; beyond, 1 x
        // 40 000: 17.2, two waves a tile 18.3)
        if (tiles < 2048 && chunks > 1) {
            red = (size_t)SCORE_WAVES * nt * 64 * (full ? 16 : 4);
            fit();
            while (ks < 8 && tiles * ks < 4096 && ks * 2 <= slice) ks *= 2;
        }
        a.slice = slice;
        a.ks = ks;
        const int64_t wgs = (tiles + SCORE_WAVES / ks - 1) / (SCORE_WAVES / ks);
        const unsigned grid = (unsigned)(wgs < 256 ? wgs : 256);
        const size_t lds = (size_t)SCORE_WAVES * SCORE_STRIP + (size_t)lrows * (slice * 256 + SCORE_PAD(full)) + red;
        hipError_t e;
        if (group == 32) e = bf ? scores_launch<true, 32>(a, mt, grid, lds, st) : scores_launch<false, 32>(a, mt, grid, lds, st);
        else if (group == 64) e = bf ? scores_launch<true, 64>(a, mt, grid, lds, st) : scores_launch<false, 64>(a, mt, grid, lds, st);
        else e = bf ? scores_launch<true, 128>(a, mt, grid, lds, st) : scores_launch<false, 128>(a, mt, grid, lds, st);
        if (e != hipSuccess) return abc_fail_hip(e, "store_scores launch");
    }
    return ABC_OK;
}
