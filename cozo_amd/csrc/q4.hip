// q4.hip -- 4-bit rows with group scales: quantising, decoding, products with queries, exhaustive k-NN (form and arithmetic:
// include/cozo_gpu.h).
#include <algorithm>
#include <cmath>

#include "call.h"
#include "distance.h"
#include "gemm_nt.h"
#include "topk.h"

using namespace czd;

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kMaxDim = 8192;

constexpr uint32_t kTile = 64;        // rows that the search looks at together

struct Rows {
    const uint8_t *codes;
    const uint16_t *scales;
    uint32_t n, dim;
    uint32_t gshift;  // log2 of the group
    uint32_t groups;  // per row
    uint32_t chunks;  // per row, of 8 elements (4 bytes of codes): groups * group / 8
};

__device__ __forceinline__ float bf16_to_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
// round to nearest even; finite input
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {
    const uint32_t u = __float_as_uint(f);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ int code_at(uint32_t w, int j) { return (int)(w << (28 - 4 * j)) >> 28; }

// 8 elements of a row (f32 or bf16) from element e0; what lies behind `dim` is 0.  `wide`: rows are 16-byte aligned
template <typename E>
__device__ __forceinline__ void load8(const E *row, uint32_t e0, uint32_t dim, bool wide, float v[8]) {
    if (wide && e0 + 8 <= dim) {
        if constexpr (sizeof(E) == 4) {
            const f32x4 a = *(const f32x4 *)(row + e0), b = *(const f32x4 *)(row + e0 + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = a[j], v[4 + j] = b[j];
        } else {
            const u32x4 a = *(const u32x4 *)(row + e0);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[2 * j] = __uint_as_float(a[j] << 16);
                v[2 * j + 1] = __uint_as_float(a[j] & 0xFFFF0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float x = 0.f;
        if (e0 + j < dim) {
            if constexpr (sizeof(E) == 4) x = row[e0 + j];
            else x = bf16_to_f32(row[e0 + j]);
        }
        v[j] = x;
    }
}

// ---- quantise --------------------------------------------------------------------------------------------------------
// HBM bound: 4 (2) bytes read and 0.53 written per element.  LPR lanes own a row, a lane 8 consecutive elements at a time (two 16-byte
// loads, one 4-byte store of codes); a group is 4 / 8 / 16 neighbouring lanes, so its maximum is 2-4 lane exchanges and never
// leaves the wave.  The squared norm is exact up to its f64 sums: a lane adds its code squares as integers.
template <typename E, int LPR>
__global__ void __launch_bounds__(256)
q4_quantize_kernel(const E *__restrict__ x, uint64_t ld, bool wide, Rows t, uint8_t *__restrict__ codes, uint16_t *__restrict__ scales,
                   float *__restrict__ sqnorms) {
    const int sub = threadIdx.x % LPR;
    const int glanes = 1 << (t.gshift - 3);
    for (uint64_t r0 = (uint64_t)blockIdx.x * (256 / LPR); r0 < t.n; r0 += (uint64_t)gridDim.x * (256 / LPR)) {
        const uint64_t r = r0 + threadIdx.x / LPR;
        const bool live = r < t.n;
        double sq = 0.0;
        bool some = false;
        for (uint32_t c0 = 0; c0 < t.chunks; c0 += LPR) {  // (uniform: the lanes of a group are active together)
            const uint32_t c = c0 + sub;
            const bool on = live && c < t.chunks;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 0.f;
            if (on) load8(x + r * ld, c * 8, t.dim, wide, v);
            float m = 0.f;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                m = fmaxf(m, fabsf(v[j]));
                bad |= !(fabsf(v[j]) < __builtin_inff());
            }
            if (bad) m = __builtin_inff();
            for (int o = 1; o < glanes; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            uint16_t sb = 0;
            float inv = 0.f;
            if (m == __builtin_inff()) {
                sb = 0x7FC0;  // NaN: the group stands for nothing
            } else if (m >= 0x1p-60f) {
                sb = f32_to_bf16(__fdiv_rn(m, 7.0f));
                inv = __fdiv_rn(1.0f, bf16_to_f32(sb));
            }
            uint32_t w = 0;
            int cc = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float q = rintf(v[j] * inv);
                q = fminf(fmaxf(q, -7.f), 7.f);
                const int k = m == __builtin_inff() ? 0 : (int)q;
                cc += k * k;
                w |= (uint32_t)(k & 15) << (4 * j);
            }
            const double s = (double)bf16_to_f32(sb);
            if (m == __builtin_inff()) sq += (double)__builtin_nanf("");
            else sq += (double)cc * (s * s);
            some |= cc != 0;
            if (on) {
                *(uint32_t *)(codes + (r * t.chunks + c) * 4) = w;
                if ((c & (glanes - 1)) == 0) scales[r * t.groups + (c >> (t.gshift - 3))] = sb;
            }
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) {
            sq += __shfl_xor(sq, o, 64);
            some |= (bool)__shfl_xor((int)some, o, 64);
        }
        if (live && sub == 0) {
            float f = (float)sq;
            if (some && f == 0.f) f = __uint_as_float(1);
            sqnorms[r] = f;
        }
    }
}

// ---- decode ----------------------------------------------------------------------------------------------------------
// HBM bound by the 4 bytes written per element; a lane writes 8 consecutive elements (two 16-byte stores when the rows allow it)
__global__ void __launch_bounds__(256)
q4_dequantize_kernel(Rows t, const uint32_t *__restrict__ rows, uint32_t m, bool wide, float *__restrict__ out) {
    const uint64_t total = (uint64_t)m * t.chunks;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t o = (uint32_t)(i / t.chunks), c = (uint32_t)(i - (uint64_t)o * t.chunks);
        const uint32_t e0 = c * 8;
        if (e0 >= t.dim) continue;
        const uint32_t r = rows ? rows[o] : o;
        float v[8];
        if (r < t.n) {
            const uint32_t w = *(const uint32_t *)(t.codes + ((uint64_t)r * t.chunks + c) * 4);
            const float s = bf16_to_f32(t.scales[(uint64_t)r * t.groups + (e0 >> t.gshift)]);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (float)code_at(w, j) * s;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __builtin_nanf("");
        }
        float *p = out + (uint64_t)o * t.dim + e0;
        if (wide) {  // dim is a multiple of 4: a lane's elements end inside the row or after its fourth
            *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]};
            if (e0 + 4 < t.dim) *(f32x4 *)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (e0 + j < t.dim) p[j] = v[j];
        }
    }
}

// ---- products on the matrix cores -------------------------------------------------------------------------------------
// A row's codes are 8-bit integers for the matrix cores after one mask per nibble (the code in a byte's upper half: 16 times it), so
// a query becomes integers too: fixed point with 31 bits below its largest element, cut into four balanced 8-bit digits.
//   v_mfma_i32_16x16x64_i8:  A (16 rows) = 4 queries x 4 digits,  B (16 columns) = 16 table rows,  64 elements at a time.
// Sums within a group are exact.  Lane l of the result holds the four digits of query l / 16 for table row l % 16: they are joined in
// the lane (two integer shifts-and-adds, two conversions, one fma), put into the sums' unit (a power of two, one multiplication) and added to
// one f32 accumulator with the lane's own row's scale.
// Rounding: 2^-31 of the query's largest element, and f32 sums over the groups.
// HBM bound up to about 16 queries: per 512 bytes of codes (16 rows x 64 elements) a wave issues 14 vector instructions and one matrix
// instruction for each 4 queries.
typedef int i32x4 __attribute__((ext_vector_type(4)));

// A query whose norm's square is below this has no score (its norm is given as NaN, and every row is looked at in f64): products with rows of 1e-15,
// the smallest whose cosine has one, would fall under the f32 range's lower end and be off by more than the score's bound says (2^-150 / 1e-15
// to 2^-20 of a norm of 2^-80).
constexpr double kLeastSquare = 0x1p-160;

constexpr int kNotFinite = -100000;  // exponent of a query that holds a NaN or an infinity

// The products of a query whose elements are below 2^e are summed in units of 2^(e - sum_exponent(e)):
//   e >= 0           2^17: a sum leaves the f32 range only 2^17 beyond the largest result
//   -17 < e < 0      2^(e + 17)
//   -90 <= e <= -17  1, the result's own
//   e < -90          2^(e + 90), so that the factor that brings a joined sum to its unit stays a normal number
// Below e = 0 no sum leaves the range: 8192 elements of 8 times the largest scale are 2^144, times 2^e.  What is lost below the range is at most
// 2^-133 of the result for each group.
__device__ __forceinline__ int sum_exponent(int e) { return e >= 0 ? e - 17 : max(min(e, -17), -90); }

// The element (of a step's 64) that byte j of lane l's 16 bytes stands for.  A lane loads 16 bytes of codes, 32 consecutive elements; lanes
// 0-31 hold a step's 64, lanes 32-63 the next step's, and a swap of half registers gives every lane 16 of either: the first or the second
// 16 of its 32.  A dword of codes unpacks into its even and then its odd elements.
__device__ __forceinline__ int element_of_byte(int l, int j) {
    return ((l >> 4) & 1) * 32 + (l >> 5) * 16 + (j & 8) + ((j & 4) ? 2 * (j & 3) + 1 : 2 * (j & 3));
}

// one workgroup per 4 queries: digits [block][step][lane][16 bytes] in the order the matrix instruction reads them, the exponent of the
// fixed point, the norm.  A fixed-point number v has the balanced digits  byte k of (v + 0x00808080), less 128 for the lower three.
__global__ void __launch_bounds__(256)
q4_digits_kernel(const float *__restrict__ q, uint32_t B, uint32_t dim, uint32_t steps, uint32_t *__restrict__ digits,
                 int *__restrict__ exponent, float *__restrict__ norm) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    uint32_t *fixed = (uint32_t *)smem_raw;  // [4][steps * 64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t b = blockIdx.x * 4 + wave, width = steps * 64;
    {   // a wave per query
        const float *row = q + (uint64_t)min(b, B - 1) * dim;
        float m = 0.f;
        double s2 = 0.0;
        bool bad = false;
        for (uint32_t i = lane; i < width; i += 64) {
            const float v = i < dim ? row[i] : 0.f;
            fixed[wave * width + i] = __float_as_uint(v);
            m = fmaxf(m, fabsf(v));
            bad |= !(fabsf(v) < __builtin_inff());
            s2 = fma((double)v, (double)v, s2);
        }
        if (bad) m = __builtin_inff();
        for (int o = 32; o; o >>= 1) {
            m = fmaxf(m, __shfl_xor(m, o, 64));
            s2 += __shfl_xor(s2, o, 64);
        }
        int e = 0;
        if (m == __builtin_inff()) e = kNotFinite;
        else if (m > 0.f) (void)frexpf(m, &e);
        if (lane == 0 && b < B) {
            exponent[b] = e;
            if (norm) norm[b] = e == kNotFinite || s2 < kLeastSquare ? __builtin_nanf("") : __double2float_ru(sqrt(s2));
        }
        const bool on = b < B && e != kNotFinite;
        for (uint32_t i = lane; i < width; i += 64) {
            const float v = __uint_as_float(fixed[wave * width + i]);
            // (a power of two: exact, or below the half step that is rounded away)
            fixed[wave * width + i] = on ? ((uint32_t)(int)rintf(ldexpf(v, 30 - e)) + 0x00808080u) ^ 0x00808080u : 0u;
        }
    }
    __syncthreads();
    // a thread makes the 4 bytes of one dword: step, lane of the instruction, dword
    for (uint32_t i = threadIdx.x; i < steps * 256; i += 256) {
        const uint32_t step = i >> 8, l = (i >> 2) & 63, w = i & 3;
        const uint32_t row = l & 15, shift = (row & 3) * 8;
        const uint32_t *f = fixed + (row >> 2) * width + step * 64;
        uint32_t out = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) out |= ((f[element_of_byte(l, 4 * w + j)] >> shift) & 255u) << (8 * j);
        digits[(uint64_t)blockIdx.x * steps * 256 + i] = out;
    }
}

// RT x 16 rows and CT x 4 queries to a wave; the digits of the workgroup's queries stay in LDS while its waves go over the table.
// A batch is 256 elements of each row, whole 128-byte lines (read 64 bytes at a time, the lines of 16 waves do not stay in the L1:
// 1.15 ms instead of 0.76 for one query against 10M x 768, 5.4 TB/s), and loads run one batch ahead, across tiles.  SW: a batch's scales of a row come in one load.
template <int RT, int CT, int GS, bool SW>
struct Product {
    static constexpr int KU = 4;                     // steps (64 elements) of a batch
    static constexpr int SC = GS == 5 ? 8 : GS == 6 ? 4 : 2;  // scales of a batch
    struct Batch {
        u32x4 w[KU / 2][RT];
        uint32_t s[RT][SC / 2];  // two scales to a word
    };
    float acc[RT][CT];

    __device__ __forceinline__ static void load(Batch &x, const Rows &t, uint64_t row0, uint32_t k) {
        const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
        const uint32_t row_bytes = t.chunks * 4;
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const uint64_t r = min(row0 + 16 * i + col, (uint64_t)t.n - 1);  // (rows past the last one: the caller drops them)
            const uint8_t *c = t.codes + r * row_bytes;
            const uint16_t *s = t.scales + r * t.groups;
#pragma unroll
            for (int u = 0; u < KU / 2; u++)  // (where a row ends inside the batch the digits are 0 or the step is not taken)
                x.w[u][i] = *(const u32x4 *)(c + min((k + 2 * u) * 32 + kg * 16, row_bytes - 16));
            const uint32_t g0 = GS == 5 ? k * 2 : GS == 6 ? k : k >> 1;
            if constexpr (SW) {
                if constexpr (SC == 8) *(u32x4 *)x.s[i] = *(const u32x4 *)(s + g0);
                else if constexpr (SC == 4) *(u32x2 *)x.s[i] = *(const u32x2 *)(s + g0);
                else x.s[i][0] = *(const uint32_t *)(s + g0);
            } else {
#pragma unroll
                for (int h = 0; h < SC / 2; h++) {
                    const uint32_t a = s[min(g0 + 2 * h, t.groups - 1)], b = s[min(g0 + 2 * h + 1, t.groups - 1)];
                    x.s[i][h] = a | (b << 16);
                }
            }
        }
    }
    __device__ __forceinline__ static float scale(const Batch &x, int i, int h) {
        const uint32_t w = x.s[i][h >> 1];
        return __uint_as_float((h & 1) ? w & 0xFFFF0000u : w << 16);
    }
    __device__ __forceinline__ static float join(const i32x4 &d) {
        const int hi = (d[3] << 8) + d[2], lo = (d[1] << 8) + d[0];  // (a digit's sum is at most 16 * 8 * 128 * 128 = 2^21)
        return fmaf((float)hi, 65536.f, (float)lo);
    }
    __device__ __forceinline__ static i32x4 unpack(uint32_t w0, uint32_t w1) {
        return i32x4{(int)((w0 << 4) & 0xF0F0F0F0u), (int)(w0 & 0xF0F0F0F0u), (int)((w1 << 4) & 0xF0F0F0F0u), (int)(w1 & 0xF0F0F0F0u)};
    }
    // UNIT: joined sums are multiplied by the query's unit[c] first
    template <bool UNIT>
    __device__ __forceinline__ void work(const Batch &x, const u32x4 *lds, uint32_t k, uint32_t steps, const float (&unit)[CT]) {
        auto add = [&](int i, int c, const i32x4 &d, float s) { acc[i][c] = fmaf(UNIT ? join(d) * unit[c] : join(d), s, acc[i][c]); };
        const int lane = threadIdx.x & 63;
        i32x4 open[RT][CT];  // (a group of 128 is two steps of one batch)
#pragma unroll
        for (int u = 0; u < KU; u++) {
            if (k + u >= steps) break;  // (uniform)
            i32x4 b[RT];
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const u32x4 w = x.w[u / 2][i];
                const u32x2 p = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), q = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                b[i] = unpack(p[u & 1], q[u & 1]);
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const u32x4 a4 = lds[(c * steps + k + u) * 64 + lane];
                const i32x4 a = {(int)a4[0], (int)a4[1], (int)a4[2], (int)a4[3]}, none = {0, 0, 0, 0};
                if constexpr (GS == 5) {  // two groups in a step: lanes 0-15 and 32-47 hold the elements of the first
                    const bool first = (lane & 16) == 0;
                    const i32x4 a0 = first ? a : none, a1 = first ? none : a;
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        const i32x4 d0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b[i], none, 0, 0, 0);
                        const i32x4 d1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b[i], none, 0, 0, 0);
                        add(i, c, d0, scale(x, i, 2 * u));
                        add(i, c, d1, scale(x, i, 2 * u + 1));
                    }
                } else if constexpr (GS == 6) {
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        const i32x4 d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b[i], none, 0, 0, 0);
                        add(i, c, d, scale(x, i, u));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        open[i][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b[i], (u & 1) ? open[i][c] : none, 0, 0, 0);
                        if (u & 1) add(i, c, open[i][c], scale(x, i, u / 2));
                    }
                }
            }
        }
    }
};

// score of a row for the search: larger is nearer, in f32; a row whose score says nothing reliable is as near as can be (its tile is
// looked at in f64), a row of zeros has no cosine
__device__ __forceinline__ float score_of(int metric, float dot, float sq) {
    float v = dot;
    if (metric == CZ_COSINE) {
        if (sq == 0.f) return -__builtin_inff();
        v = dot * rsqrtf(sq);
    } else if (metric == CZ_L2) {
        v = fmaf(2.f, dot, -sq);
    }
    const bool sure = sq < __builtin_inff() && (sq >= 1e-30f || metric != CZ_COSINE) && fabsf(v) < __builtin_inff();
    return sure ? v : __builtin_inff();
}
// how far a score may be off: `c` of |q| |x| (the product), for L2 the norm's and the difference's rounding, and what the lower end of
// the f32 range cuts off
__device__ __forceinline__ float score_error(int metric, float c, float qnorm, float xnorm) {
    if (metric == CZ_COSINE) return c * qnorm + 0x1p-140f;
    if (metric == CZ_IP) return c * qnorm * xnorm + 0x1p-140f;
    return 2.f * c * qnorm * xnorm + 0x1p-22f * xnorm * xnorm + 0x1p-140f;
}

// what some row of a tile is sure to reach; a tile with a row whose score says nothing is sure of nothing
__device__ __forceinline__ float sure_score(int metric, float c, float qnorm, float xnorm, float top) {
    return top < __builtin_inff() ? top - score_error(metric, c, qnorm, xnorm) : -__builtin_inff();
}

// Products of these norms, or what a score makes of them, may pass the f32 range: no score then says anything (one that was to be near may have
// become minus infinity).  A cosine's score is at most the query's norm.
__device__ __forceinline__ bool may_overflow(int metric, float qnorm, float xnorm) {
    return metric != CZ_COSINE && !((metric == CZ_L2 ? fmaf(2.f, qnorm, xnorm) : qnorm) * xnorm < 0x1p126f);
}

struct Near {              // what the search takes from the product kernels instead of the products
    int metric;
    const float *sqnorms;
    float err;             // c of score_error
    const float *qnorm;    // [B]
    float *tile_score;     // [B][n_tiles] largest score of a tile
    float *tile_norm;      // [n_tiles] largest norm of a tile's rows
    float *best;           // [B][n_best] what some row of a wave's tiles is sure to reach
    uint32_t n_tiles, n_best;
};

// workgroups of a CU (of 4 waves, one to a SIMD): what the registers of CT accumulators and two batches leave room for
constexpr int residents(int ct, int gshift) { return ct == 1 ? (gshift == 5 ? 3 : 4) : ct == 2 && gshift != 5 ? 3 : 2; }

template <int CT, int GS, bool SW, bool NEAR>
__global__ void __launch_bounds__(256, residents(CT, GS))
q4_product_kernel(Rows t, const u32x4 *__restrict__ digits, const int *__restrict__ exponent, uint32_t B, uint32_t steps, float *__restrict__ out,
                  Near near) {
    constexpr int RT = 4;
    static_assert(RT * 16 == kTile, "a wave's rows are a tile of the search");
    typedef Product<RT, CT, GS, SW> P;
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    u32x4 *lds = (u32x4 *)smem_raw;  // [CT][steps][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15;
    const uint32_t c0 = blockIdx.y * CT, blocks4 = (B + 3) / 4;
    for (uint32_t i = threadIdx.x; i < CT * steps * 64; i += 256) {
        const uint32_t c = c0 + i / (steps * 64);
        lds[i] = c < blocks4 ? digits[(uint64_t)c0 * steps * 64 + i] : u32x4{0, 0, 0, 0};
    }
    int ex[CT];  // of a sum's unit
    float best[CT], qn[CT], unit[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const uint32_t b = (c0 + c) * 4 + (lane >> 4);
        const int e = b < B ? exponent[b] : 0;
        // a joined sum is in units of 2^(e - 34): the fixed point's 30 bits and the codes' 4.  The search keeps that (a score beyond the
        // range says nothing, and its tile is looked at)
        ex[c] = e == kNotFinite ? e : NEAR ? e - 34 : e - sum_exponent(e);
        unit[c] = NEAR || e == kNotFinite ? 1.f : ldexpf(1.f, sum_exponent(e) - 34);
        best[c] = -__builtin_inff();
        qn[c] = NEAR && b < B ? near.qnorm[b] : 0.f;
    }
    __syncthreads();
    const uint64_t n_tiles = ((uint64_t)t.n + kTile - 1) / kTile, stride = (uint64_t)gridDim.x * 4;
    uint64_t tile = (uint64_t)blockIdx.x * 4 + wave;
    typename P::Batch cur, nxt;
    P p;
    if (tile < n_tiles) P::load(cur, t, tile * kTile, 0);
    while (tile < n_tiles) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int c = 0; c < CT; c++) p.acc[i][c] = 0.f;
        for (uint32_t k = 0; k < steps; k += P::KU) {
            const bool more = k + P::KU < steps;
            const uint64_t nt = more ? tile : tile + stride;
            if (nt < n_tiles) P::load(nxt, t, nt * kTile, more ? k + P::KU : 0);
            p.template work<!NEAR>(cur, lds, k, steps, unit);
            cur = nxt;
        }
        float sq[RT], xn = 0.f;
        if constexpr (NEAR) {
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const uint64_t r = tile * kTile + 16 * i + col;
                sq[i] = r < t.n ? near.sqnorms[r] : 0.f;
                if (sq[i] < __builtin_inff()) xn = fmaxf(xn, sq[i]);
            }
            for (int o = 1; o < 16; o <<= 1) xn = fmaxf(xn, __shfl_xor(xn, o, 64));
            xn = sqrtf(xn) * 1.0001f + 1e-22f;  // (a square may be rounded off the f32 range's lower end)
            if (blockIdx.y == 0 && lane == 0) near.tile_norm[tile] = xn;
        }
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const uint32_t b = (c0 + c) * 4 + (lane >> 4);
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const uint64_t r = tile * kTile + 16 * i + col;
                const float v = ex[c] == kNotFinite ? __builtin_nanf("") : ldexpf(p.acc[i][c], ex[c]);
                if constexpr (NEAR) {
                    if (r < t.n) top = fmaxf(top, score_of(near.metric, v, sq[i]));
                } else {
                    if (r < t.n && b < B) out[(uint64_t)b * t.n + r] = v;
                }
            }
            if constexpr (NEAR) {
                for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
                if (b < B && col == 0) near.tile_score[(uint64_t)b * near.n_tiles + tile] = top;
                best[c] = fmaxf(best[c], sure_score(near.metric, near.err, qn[c], xn, top));
            }
        }
        tile += stride;
    }
    if constexpr (NEAR) {
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const uint32_t b = (c0 + c) * 4 + (lane >> 4);
            if (b < B && col == 0) near.best[(uint64_t)b * near.n_best + blockIdx.x * 4 + wave] = best[c];
        }
    }
}

// ---- scores of many queries: an f16 matrix product ----------------------------------------------------------------------
// For a large batch the search's scores come from a product in f16 (the f64 distances decide, so a score only has to be within a bound that
// is known): a row's codes become f16 once per 256 queries instead of once per 4, and one matrix instruction does what the digits take four
// for.  Both sides are scaled by a power of two to a norm of at most 2^8, so that nothing that matters is below f16's normal range:
//   error <= |q| |x| (2^-11 of rounding the query + sqrt(dim) 2^-20 of what is flushed + dim 2^-24 of the f32 sums)
// The loop is that of gemm_nt.h with the table's side made in registers: 16 bytes of codes (32 elements) a thread and step, loaded two steps
// ahead, four packed f16 operations per 4 elements.  1M x 768, 1024 queries: 1.9 ms, 0.83 PFLOP/s; the same loop over bf16 rows runs at 1.05.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// the element (of 8) at each place of a 16-byte piece: a dword's nibbles are taken 16 bits apart
__device__ __forceinline__ uint32_t element_of_place(uint32_t p) { return (p >> 1) + (p & 1) * 4; }

// one wave per query: its f16 form [steps * 64] in the pieces' order, its exponent (value = form * 2^exponent) and norm
__global__ void __launch_bounds__(256)
q4_halves_kernel(const float *__restrict__ q, uint32_t B, uint32_t dim, uint32_t steps, _Float16 *__restrict__ out, int *__restrict__ exponent,
                 float *__restrict__ norm) {
    const uint32_t b = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, width = steps * 64;
    if (b >= B) return;
    const float *row = q + (uint64_t)b * dim;
    double s2 = 0.0;
    for (uint32_t i = lane; i < dim; i += 64) s2 = fma((double)row[i], (double)row[i], s2);
    for (int o = 32; o; o >>= 1) s2 += __shfl_xor(s2, o, 64);
    // (beyond 2^96, an infinity or NaN among it: no score either)
    const bool fine = s2 >= kLeastSquare && s2 < 0x1p192;
    int e = 0;
    if (fine) {
        (void)frexp(s2, &e);
        e = ((e + 1) >> 1) - 8;  // norm < 2^(e + 8)
    }
    if (lane == 0) {
        exponent[b] = e;
        norm[b] = fine ? __double2float_ru(sqrt(s2)) : __builtin_nanf("");
    }
    for (uint32_t i = lane; i < width; i += 64) {
        const uint32_t el = (i & ~7u) + element_of_place(i & 7);
        out[(uint64_t)b * width + i] = fine && el < dim ? (_Float16)ldexpf(row[el], -e) : (_Float16)0.f;
    }
}

// largest norm of each tile's rows (those that are finite)
__global__ void __launch_bounds__(256) q4_tile_norm_kernel(const float *__restrict__ sqnorms, uint32_t n, float *__restrict__ tile_norm) {
    const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6), r = tile * kTile + (threadIdx.x & 63);
    if (tile * kTile >= n) return;
    const float sq = r < n ? sqnorms[r] : 0.f;
    float x = sq < __builtin_inff() ? sq : 0.f;
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    if ((threadIdx.x & 63) == 0) tile_norm[tile] = sqrtf(x) * 1.0001f + 1e-22f;
}

// scores [tile][ldb] of 64-row tiles: a workgroup keeps BN queries and goes over its stretch of the table, BM rows at a time
template <class G, int GS>
__global__ void __launch_bounds__(G::kThreads)
q4_scores_kernel(Rows t, gemm::Operand Q, const int *__restrict__ exponent, uint32_t steps, Near near, float *__restrict__ score, uint32_t ldb,
                 uint32_t n_blocks, uint32_t blocks_per_part) {
    constexpr int BM = G::BM, BN = G::BN, TW = G::MT / 2;  // search tiles of a wave
    static_assert(G::kThreads == 2 * BM, "two threads make a row of a step");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float2 *rowf = (float2 *)(lds + G::kLds);  // [BM] factor and addend that turn a product into a score
    const int tid = threadIdx.x, lane = tid & 63, mine = tid >> 1, half = tid & 1;
    const uint32_t qt = (Q.rows + BN - 1) / BN, at = gemm::place_in_order();
    const uint32_t n0 = at % qt * BN, part = at / qt;
    const uint32_t k0 = part * blocks_per_part, k1 = min(n_blocks, k0 + blocks_per_part);
    const uint32_t row_bytes = t.chunks * 4;
    // of the two waves on a SIMD one makes its rows before and one after its matrix instructions, so that these do not wait for both
    const bool early = tid < 256;
    float best[G::NT], qn[G::NT];
    int qe[G::NT];
#pragma unroll
    for (int j = 0; j < G::NT; j++) {
        const uint32_t b = min(n0 + G::wave_col() + j * 32 + (lane & 31), Q.rows - 1);
        best[j] = -__builtin_inff();
        qn[j] = near.qnorm[b];
        qe[j] = exponent[b];
    }
    const typename G::CopiesB src(Q, n0);
#pragma unroll 1
    for (uint32_t blk = k0; blk < k1; blk++) {
        const uint64_t r = (uint64_t)blk * BM + mine, safe = min(r, (uint64_t)t.n - 1);
        const uint8_t *codes = t.codes + safe * row_bytes;
        const uint16_t *scales = t.scales + safe * t.groups;
        u32x4 w;
        uint16_t sb;
        auto load = [&](uint32_t s) {
            w = *(const u32x4 *)(codes + min(s * 32 + half * 16, row_bytes - 16));  // (past the row's end: times zeros of the query)
            sb = scales[min(GS == 5 ? 2 * s + half : GS == 6 ? s : s >> 1, t.groups - 1)];
        };
        load(0);
        G::copy(src, 0, lds + BM * 128);
        const float sq = near.sqnorms[safe];
        int e = 0;
        const bool finite = sq < __builtin_inff();
        if (finite && sq > 0.f) {
            (void)frexpf(sq, &e);
            e = ((e + 1) >> 1) - 8;
        }
        const float down = finite ? ldexpf(1.f, -e) : 0.f;  // (a row that is not finite: zeros, it is looked at anyway)
        if (half == 0) {
            float2 f = make_float2(0.f, -__builtin_inff());
            if (r < t.n) {
                const bool unsure = !finite || (near.metric == CZ_COSINE && sq > 0.f && sq < 1e-30f);
                if (unsure) f.y = __builtin_inff();
                else if (near.metric == CZ_COSINE) {
                    if (sq > 0.f) f = make_float2(ldexpf(rsqrtf(sq), e), 0.f);
                } else {
                    f = near.metric == CZ_IP ? make_float2(ldexpf(1.f, e), 0.f) : make_float2(ldexpf(2.f, e), -sq);
                }
            }
            rowf[mine] = f;
        }
        auto store = [&](char *to) {  // the loaded 32 elements as f16, at their places of the operand's row
            // (a group with a code that counts has a scale of at most the row's norm, 2^8 here; that of a group of zeros, which the norm does not
            // bound, is cut, so that none of its 16 codes, the padding's among them, makes an infinity that a zero would turn into NaN)
            const _Float16 s = (_Float16)fminf(bf16_to_f32(sb) * down, 4096.f);
            const f16x2 s2 = {finite ? s : (_Float16)0.f, finite ? s : (_Float16)0.f}, off = {(_Float16)1032.f, (_Float16)1032.f};
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const uint32_t u = w[d] ^ 0x88888888u;
                u32x4 o;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const f16x2 h = __builtin_bit_cast(f16x2, ((u >> (4 * x)) & 0x000F000Fu) | 0x64006400u) - off;  // 1024 + code + 8 - 1032
                    o[x] = __builtin_bit_cast(uint32_t, h * s2);
                }
                *(u32x4 *)(to + mine * 128 + (((half * 4 + d) ^ ((mine >> 1) & 7)) * 16)) = o;
            }
        };
        store(lds);
        if (steps > 1) load(1);
        G g;
        g.zero();
#pragma unroll 1
        for (uint32_t s = 0; s < steps; s++) {
            char *cur = lds + (s & 1) * G::kBytes, *nxt = lds + (~s & 1) * G::kBytes;
            // this step's copies are in LDS; the two loads behind them (codes and scale of the step after) may still be on their way
            // (__syncthreads would wait for all of them)
            if (s > 0 && s + 1 < steps) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (s + 1 < steps) {
                if (early) store(nxt);
                asm volatile("" ::: "memory");  // (in this order: the wait above counts on it)
                G::copy(src, s + 1, nxt + BM * 128);
                asm volatile("" ::: "memory");
                if (early && s + 2 < steps) load(s + 2);
            }
            g.template step<>(cur);
            if (!early && s + 1 < steps) {
                store(nxt);
                if (s + 2 < steps) load(s + 2);
            }
        }
        float top[G::NT][TW];
#pragma unroll
        for (int j = 0; j < G::NT; j++)
#pragma unroll
            for (int x = 0; x < TW; x++) top[j][x] = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < G::MT; i++)
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                float2 f[4];
#pragma unroll
                for (int x = 0; x < 4; x++) f[x] = rowf[G::wave_row() + i * 32 + 8 * r4 + 4 * (lane >> 5) + x];
#pragma unroll
                for (int j = 0; j < G::NT; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        top[j][i / 2] = fmaxf(top[j][i / 2], fmaf(ldexpf(g.acc[i][j][4 * r4 + x], qe[j]), f[x].x, f[x].y));
            }
#pragma unroll
        for (int x = 0; x < TW; x++) {
            const uint32_t tile = blk * (BM / kTile) + G::wave_row() / kTile + x;
            if (tile >= near.n_tiles) break;  // (uniform)
            const float xn = near.tile_norm[tile];
#pragma unroll
            for (int j = 0; j < G::NT; j++) {
                const uint32_t b = n0 + G::wave_col() + j * 32 + (lane & 31);
                float v = fmaxf(top[j][x], __shfl_xor(top[j][x], 32, 64));
                if (may_overflow(near.metric, qn[j], xn)) v = __builtin_inff();
                if (b < Q.rows && lane < 32) score[(uint64_t)tile * ldb + b] = v;
                best[j] = fmaxf(best[j], sure_score(near.metric, near.err, qn[j], xn, v));
            }
        }
        __syncthreads();  // LDS is free for the next rows
    }
#pragma unroll
    for (int j = 0; j < G::NT; j++) {
        const uint32_t b = n0 + G::wave_col() + j * 32 + (lane & 31);
        if (b < Q.rows && lane < 32) near.best[(uint64_t)b * near.n_best + part * G::WM + (tid >> 6) / G::WN] = best[j];
    }
}

// [rows][ld] -> [cols][rows], 64 x 64 through LDS
__global__ void __launch_bounds__(256)
q4_turn_kernel(const float *__restrict__ x, uint32_t rows, uint32_t cols, uint32_t ld, float *__restrict__ out) {
    __shared__ float tile[64][65];
    const uint32_t r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, c = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (uint32_t i = w; i < 64; i += 4)
        if (r0 + i < rows && c0 + c < cols) tile[i][c] = x[(uint64_t)(r0 + i) * ld + c0 + c];
    __syncthreads();
    for (uint32_t i = w; i < 64; i += 4)
        if (c0 + i < cols && r0 + c < rows) out[(uint64_t)(c0 + i) * rows + r0 + c] = tile[c][i];
}

// order-preserving u32 of an f32; NaN as -inf
__device__ __forceinline__ uint32_t order_of(float f) {
    if (f != f) f = -__builtin_inff();
    const uint32_t u = __float_as_uint(f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// need[b]: a score that k rows are sure to reach (limit[b]: the distance that goes with it) = the k-th largest of what `n` waves (or, where there are too few of them, tiles) are
// sure to hold, each a row of its own.  Radix selection, 8 bits at a time.  -inf (every row is looked at) when there are fewer than k or the
// k-th is not finite.
__global__ void __launch_bounds__(1024)
q4_need_kernel(Near near, bool by_tile, uint32_t k, float *__restrict__ need, double *__restrict__ limit) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sel[2];
    const uint32_t b = blockIdx.x, n = by_tile ? near.n_tiles : near.n_best;
    const float *v = (by_tile ? near.tile_score : near.best) + (uint64_t)b * n;
    const float qn = near.qnorm[b];
    if (n < k) {
        if (threadIdx.x == 0) {
            need[b] = -__builtin_inff();
            limit[b] = __builtin_inf();
        }
        return;
    }
    constexpr int R = 16;  // values a thread keeps; more are read again for each 8 bits
    uint32_t kept[R];
    auto value = [&](uint32_t i) { return order_of(by_tile ? sure_score(near.metric, near.err, qn, near.tile_norm[i], v[i]) : v[i]); };
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint32_t i = threadIdx.x + r * 1024;
        kept[r] = i < n ? value(i) : 0u;
    }
    uint32_t prefix = 0, left = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        auto count = [&](uint32_t o) {
            if (shift == 24 || (o >> (shift + 8)) == prefix) atomicAdd(&hist[(o >> shift) & 255], 1u);
        };
#pragma unroll
        for (int r = 0; r < R; r++)
            if (threadIdx.x + r * 1024 < n) count(kept[r]);
        for (uint32_t i = threadIdx.x + R * 1024; i < n; i += 1024) count(value(i));
        __syncthreads();
        if (threadIdx.x < 64) {  // suffix sums over 256 bins, 4 to a lane, from the top
            const int lane = threadIdx.x;
            uint32_t h[4], mine = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) mine += h[j] = hist[255 - (4 * lane + j)];
            uint32_t run = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t up = __shfl_up(run, o, 64);
                if (lane >= o) run += up;
            }
            uint32_t before = run - mine;
            if (before < left && left <= run) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (before < left && left <= before + h[j]) {
                        sel[0] = 255 - (4 * lane + j);
                        sel[1] = left - before;
                    }
                    before += h[j];
                }
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | sel[0];
        left = sel[1];
    }
    if (threadIdx.x == 0) {
        const float f = __uint_as_float((prefix >> 31) ? (prefix & 0x7FFFFFFFu) : ~prefix);
        const bool some = fabsf(f) < __builtin_inff();
        need[b] = some ? f : -__builtin_inff();
        // a row that k others are nearer than: its distance, with 1e-6 of what it is made of to spare for the arithmetic in between
        const double q = qn, s = f;
        double d = near.metric == CZ_COSINE ? 1.0 - s / q + 1e-6 * fabs(s / q) : near.metric == CZ_IP ? 1.0 - s + 1e-6 * fabs(s) : q * q - s + 1e-6 * (q * q + fabs(s));
        d += 1e-9 * fabs(d) + 1e-12 * (near.metric != CZ_L2);
        limit[b] = some && d == d ? d : __builtin_inf();
    }
}

// ---- exact k-NN ------------------------------------------------------------------------------------------------------
// the f64 distances of U rows from the query in LDS, by LPR neighbouring lanes (every lane returns them).  A code times an f32 is exact in
// f64; a lane's 8 codes share a scale, so it is applied once.  The lanes' sums are joined by a fixed butterfly, so equal rows have equal bits.
template <int LPR, int U>
__device__ __forceinline__ void row_distances(int metric, const Rows &t, const uint32_t (&r)[U], int sub, const double *q, double qq, double (&out)[U]) {
    double a[U], x2[U];
#pragma unroll
    for (int u = 0; u < U; u++) a[u] = x2[u] = 0.0;
    for (uint32_t c = sub; c < t.chunks; c += LPR) {
        uint32_t w[U];
        double s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            w[u] = *(const uint32_t *)(t.codes + ((uint64_t)r[u] * t.chunks + c) * 4);
            s[u] = (double)bf16_to_f32(t.scales[(uint64_t)r[u] * t.groups + ((c * 8) >> t.gshift)]);
        }
        const double *qc = q + c * 8;
        const int left = min(8, (int)t.dim - (int)(c * 8));  // (the last group's padding)
        if (left < 8)
#pragma unroll
            for (int u = 0; u < U; u++) w[u] &= left > 0 ? (1u << (4 * left)) - 1u : 0u;
        if (metric == CZ_L2) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const double qv = qc[j];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const double d = fma((double)code_at(w[u], j), -s[u], qv);
                    // (past the last element the code is 0 and so is the query)
                    a[u] = fma(d, d, a[u]);
                }
            }
        } else {
            double p[U];
            int cc[U];
#pragma unroll
            for (int u = 0; u < U; u++) p[u] = 0.0, cc[u] = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const double qv = qc[j];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int k = code_at(w[u], j);
                    p[u] = fma((double)k, qv, p[u]);
                    cc[u] += k * k;
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                a[u] = fma(p[u], s[u], a[u]);
                x2[u] = fma((double)cc[u], s[u] * s[u], x2[u]);
            }
        }
    }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1)
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] += __shfl_xor(a[u], o, 64);
            x2[u] += __shfl_xor(x2[u], o, 64);
        }
#pragma unroll
    for (int u = 0; u < U; u++) out[u] = metric == CZ_L2 ? a[u] : metric == CZ_COSINE ? 1.0 - a[u] / sqrt(qq * x2[u]) : 1.0 - a[u];
}

// bkey / bid[0 .. nb): a batch of up to 256 entries, no two of one id; tkey / tid_[0 .. tcnt): the list, ascending by (key, id), at most k.
// Every entry's rank is counted, without a branch, so that the LDS reads of the count run ahead: 3 us for a full batch.  Returns the new
// length (uniform); starts and ends with a barrier.
__device__ __forceinline__ int merge_batch(int nb, const uint64_t *bkey, const uint32_t *bid, uint64_t *tkey, uint32_t *tid_, int tcnt, int k) {
    const int tid = threadIdx.x;
    __syncthreads();
    auto before = [&](uint64_t key, uint32_t id) {
        int c = 0;
#pragma unroll 8
        for (int t = 0; t < nb; t++) {
            const uint64_t o = bkey[t];
            c += (int)((o < key) | ((o == key) & (bid[t] < id)));
        }
        return c;
    };
    uint64_t mk = 0, wk[4];
    uint32_t mi = CZ_NONE, wi[4];
    int at = k, wat[4];
    if (tid < nb) {
        mk = bkey[tid];
        mi = bid[tid];
        int lo = 0, hi = tcnt;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (czh::key_lt(tkey[mid], tid_[mid], mk, mi)) lo = mid + 1;
            else hi = mid;
        }
        at = lo + before(mk, mi);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {  // (k <= 1024)
        const int j = tid + 256 * r;
        wat[r] = k;
        if (j < tcnt) {
            wk[r] = tkey[j];
            wi[r] = tid_[j];
            wat[r] = j + before(wk[r], wi[r]);
        }
    }
    __syncthreads();
    if (at < k) {
        tkey[at] = mk;
        tid_[at] = mi;
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (wat[r] < k) {
            tkey[wat[r]] = wk[r];
            tid_[wat[r]] = wi[r];
        }
    __syncthreads();
    return min(k, tcnt + nb);
}

// the tiles that a search still has to look at in f64: those whose best score could reach what k rows are sure to reach
struct Candidates {
    const float *tile_score;  // [B][n_tiles], or null: all tiles
    const float *tile_norm;   // [n_tiles]
    const float *qnorm;       // [B]
    const float *need;        // [B]
    const double *limit;      // [B]
    float err;
};

// per (chunk of tiles, query): the k nearest rows of the chunk's candidate tiles as a sorted partial list
template <int LPR>
__global__ void __launch_bounds__(256, 3)
q4_scan_kernel(int metric, Rows t, const float *__restrict__ queries, uint32_t k, uint32_t tiles_per_chunk, Candidates cand,
               uint64_t *__restrict__ part_key, uint32_t *__restrict__ part_id, uint32_t *__restrict__ part_count) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    double *q = (double *)smem_raw;               // [chunks * 8]
    uint64_t *bkey = (uint64_t *)(q + t.chunks * 8);  // [256]
    uint64_t *tkey = bkey + 256;                  // [k]
    double *red = (double *)(tkey + k);           // [4]
    uint32_t *bid = (uint32_t *)(red + 4);        // [256]
    uint32_t *tid_ = bid + 256;                   // [k]
    uint32_t *list = tid_ + k;                    // [1024] candidate tiles
    uint32_t *cnt = list + 1024;                  // [5]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = tid % LPR;
    const uint32_t b = blockIdx.y;
    const uint32_t n_tiles = (uint32_t)(((uint64_t)t.n + kTile - 1) / kTile);
    const uint32_t t0 = blockIdx.x * tiles_per_chunk, t1 = (uint32_t)min((uint64_t)n_tiles, (uint64_t)t0 + tiles_per_chunk);
    const float need = cand.tile_score ? cand.need[b] : 0.f, qn = cand.tile_score ? cand.qnorm[b] : 0.f;
    const double limit = cand.tile_score ? cand.limit[b] : __builtin_inf();
    double qq = 0.0;
    bool ready = false;
    int tcnt = 0;
    if (tid == 0) cnt[4] = 0;  // rows in the batch
    for (uint32_t tb = t0; tb < t1; tb += 1024) {
        unsigned long long m[4];
        uint32_t at = 0, total = 0;
        bool want[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t tile = tb + 256 * i + tid;
            want[i] = tile < t1;
            if (want[i] && cand.tile_score) {
                const float s = cand.tile_score[(uint64_t)b * n_tiles + tile];
                want[i] = !(s + score_error(metric, cand.err, qn, cand.tile_norm[tile]) < need);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            m[i] = __ballot(want[i]);
            total += __popcll(m[i]);
        }
        if (lane == 0) cnt[wave] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            if (w < wave) at += cnt[w];
            total += cnt[w];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (want[i]) list[at + __popcll(m[i] & ((1ull << lane) - 1ull))] = tb + 256 * i + tid;
            at += __popcll(m[i]);
        }
        __syncthreads();
        if (total && !ready) {  // the query, once there is something to look at
            for (uint32_t i = tid; i < t.chunks * 8; i += 256) {
                const double v = i < t.dim ? (double)queries[(uint64_t)b * t.dim + i] : 0.0;
                q[i] = v;
                qq = fma(v, v, qq);
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) qq += __shfl_xor(qq, o, 64);
            if (lane == 0) red[wave] = qq;
            __syncthreads();
            qq = (red[0] + red[1]) + (red[2] + red[3]);
            ready = true;
        }
        constexpr int U = 4, AT = 256 / LPR;  // rows of a lane group at a time, lane groups: 16 to 256 rows
        const uint32_t rows = total * kTile;
        for (uint32_t s0 = 0; s0 < rows; s0 += U * AT) {
            uint32_t r[U];
            double d[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t slot = min(s0 + u * AT + tid / LPR, rows - 1);
                r[u] = (uint32_t)min((uint64_t)list[slot / kTile] * kTile + slot % kTile, (uint64_t)t.n - 1);
            }
            const uint32_t have = cnt[4];
            row_distances<LPR, U>(metric, t, r, sub, q, qq, d);
            __syncthreads();  // (everyone has read it)
            if (have + U * AT > 256) {
                tcnt = merge_batch((int)have, bkey, bid, tkey, tid_, tcnt, (int)k);
                if (tid == 0) cnt[4] = 0;
                __syncthreads();
            }
            if (sub == 0)
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint32_t slot = s0 + u * AT + tid / LPR;
                    if (slot < rows && (uint64_t)list[slot / kTile] * kTile + slot % kTile < t.n && !(d[u] > limit)) {
                        const uint64_t key = dist_key(d[u]);
                        if (tcnt < (int)k || czh::key_lt(key, r[u], tkey[k - 1], tid_[k - 1])) {
                            const uint32_t e = atomicAdd(&cnt[4], 1u);  // (the order does not matter: entries are ranked)
                            bkey[e] = key;
                            bid[e] = r[u];
                        }
                    }
                }
            __syncthreads();
        }
        __syncthreads();  // the list is free
    }
    __syncthreads();
    tcnt = merge_batch((int)cnt[4], bkey, bid, tkey, tid_, tcnt, (int)k);
    const size_t part = (size_t)b * gridDim.x + blockIdx.x;
    for (int i = tid; i < tcnt; i += 256) {
        part_key[part * k + i] = tkey[i];
        part_id[part * k + i] = tid_[i];
    }
    if (tid == 0) part_count[part] = (uint32_t)tcnt;
}

// one workgroup per query: the partial lists joined, the radius cut, the padding.  What a list takes in a full batch at a time would be merged for microseconds; the k-th
// smallest of 256 lists' heads, which k entries are sure not to be behind, leaves few to merge (one query, 157 lists: 76 -> 18 us).
constexpr size_t join_lds(size_t k) { return 256 * 24 + k * 12 + 257 * 4 + 8 * 4 + 8; }
__global__ void __launch_bounds__(256)
q4_join_kernel(const uint64_t *__restrict__ part_key, const uint32_t *__restrict__ part_id, const uint32_t *__restrict__ part_count,
               uint32_t n_parts, uint32_t k, int has_radius, double radius, uint32_t *__restrict__ out_ids, double *__restrict__ out_dist,
               uint32_t *__restrict__ out_count) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    uint64_t *bkey = (uint64_t *)smem_raw;   // [256]
    uint64_t *hkey = bkey + 256;              // [256] heads of 256 lists
    uint64_t *tkey = hkey + 256;              // [k]
    uint64_t *limit_key = tkey + k;           // [1]
    uint32_t *bid = (uint32_t *)(limit_key + 1);  // [256]
    uint32_t *hid = bid + 256;                // [256]
    uint32_t *tid_ = hid + 256;               // [k]
    uint32_t *first = tid_ + k;               // [257] entries of the parts before this one (of 256 parts at a time)
    uint32_t *ctl = first + 257;              // [0..3] waves' sums, [4] batch fill, [5] limit's id
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t b = blockIdx.x;
    int tcnt = 0, fill = 0;
    if (tid == 0) {
        ctl[4] = 0;
        ctl[5] = CZ_NONE;
        limit_key[0] = ~0ull;
    }
    for (uint32_t p0 = 0; p0 < n_parts; p0 += 256) {
        const uint32_t p = p0 + tid;
        const size_t list = (size_t)b * n_parts + p;
        const uint32_t mine = p < n_parts ? part_count[list] : 0;
        const uint64_t head_key = mine ? part_key[list * k] : ~0ull;
        const uint32_t head_id = mine ? part_id[list * k] : CZ_NONE;
        hkey[tid] = head_key;
        hid[tid] = head_id;
        uint32_t run = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(run, o, 64);
            if (lane >= o) run += up;
        }
        if (lane == 63) ctl[wave] = run;
        __syncthreads();
        for (int w = 0; w < wave; w++) run += ctl[w];
        first[tid] = run - mine;
        if (tid == 255) first[256] = run;
        if ((uint32_t)__syncthreads_count(mine != 0) >= k && mine) {
            uint32_t rank = 0;
#pragma unroll 8
            for (int t = 0; t < 256; t++) {
                const uint64_t other = hkey[t];
                rank += (uint32_t)((other < head_key) | ((other == head_key) & (hid[t] < head_id)));
            }
            if (rank == k - 1 && czh::key_lt(head_key, head_id, limit_key[0], ctl[5])) {  // (ids differ: one thread)
                limit_key[0] = head_key;
                ctl[5] = head_id;
            }
        }
        __syncthreads();
        const uint32_t total = first[256];
        const uint64_t last_key = limit_key[0];
        const uint32_t last_id = ctl[5];
        for (uint32_t e0 = 0; e0 < total; e0 += 256) {
            // entries that can still enter the list are gathered until 256 could overflow the batch
            const uint32_t e = e0 + tid;
            uint64_t key = ~0ull;
            uint32_t id = CZ_NONE;
            if (e < total) {
                uint32_t lo = 0, hi = 256;  // the part: the last one with first <= e
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (first[mid] <= e) lo = mid;
                    else hi = mid;
                }
                const size_t at = ((size_t)b * n_parts + p0 + lo) * k + (e - first[lo]);
                key = part_key[at];
                id = part_id[at];
            }
            const bool want = id != CZ_NONE && !czh::key_lt(last_key, last_id, key, id) &&
                              (tcnt < (int)k || czh::key_lt(key, id, tkey[k - 1], tid_[k - 1]));
            const int add = __syncthreads_count(want);
            if (fill + add > 256) {
                tcnt = merge_batch(fill, bkey, bid, tkey, tid_, tcnt, (int)k);
                if (tid == 0) ctl[4] = 0;
                fill = 0;
                __syncthreads();
            }
            if (want) {
                const uint32_t at = atomicAdd(&ctl[4], 1u);  // (the order within a batch does not matter: entries are ranked)
                bkey[at] = key;
                bid[at] = id;
            }
            fill += add;
        }
        __syncthreads();  // heads, sums and the limit are free
    }
    tcnt = merge_batch(fill, bkey, bid, tkey, tid_, tcnt, (int)k);
    if (tid >= 64) return;
    uint32_t done = 0;
    for (uint32_t i0 = 0; i0 < k; i0 += 64) {
        const uint32_t i = i0 + tid;
        double d = __builtin_inf();
        bool keep = (int)i < tcnt;
        if (keep) {
            d = key_dist(tkey[i]);
            keep = !(has_radius && d > radius);
        }
        const unsigned long long m = __ballot(keep);
        if (keep) {
            const uint32_t p = done + __popcll(m & ((1ull << tid) - 1ull));
            out_ids[(size_t)b * k + p] = tid_[i];
            out_dist[(size_t)b * k + p] = d;
        }
        done += __popcll(m);
    }
    for (uint32_t i = done + tid; i < k; i += 64) {
        out_ids[(size_t)b * k + i] = CZ_NONE;
        out_dist[(size_t)b * k + i] = __builtin_inf();
    }
    if (tid == 0) out_count[b] = done;
}

// ---- host side -------------------------------------------------------------------------------------------------------
// lanes that share a row: 16 (a 64-byte piece of its codes), fewer for short rows.  More spend longer on joining their sums: with 64
// the f64 distances of 1024 queries against 1M x 768 took 690 us instead of 379.
uint32_t lanes_per_row(uint32_t chunks) { return chunks <= 4 ? 4 : chunks <= 8 ? 8 : 16; }
#define CZ_Q4_LANES(LPR, CALL)      \
    switch (LPR) {                  \
        case 4: CALL(4); break;     \
        case 8: CALL(8); break;     \
        default: CALL(16); break;   \
    }

int shape_of_rows(uint32_t n, uint32_t dim, uint32_t group, Rows *t) {
    if (group != 32 && group != 64 && group != 128) return cz::set_error(CZ_E_INVALID, "group is 32, 64 or 128, not %u", group);
    if (dim == 0 || dim > kMaxDim) return cz::set_error(CZ_E_UNSUPPORTED, "dim must be in 1..%u", kMaxDim);
    if (n >= 0x80000000u) return cz::set_error(CZ_E_INVALID, "a table holds fewer than 2^31 rows");
    t->codes = nullptr;
    t->scales = nullptr;
    t->n = n;
    t->dim = dim;
    t->gshift = group == 32 ? 5 : group == 64 ? 6 : 7;
    t->groups = (dim + group - 1) / group;
    t->chunks = t->groups * (group / 8);
    return CZ_OK;
}
size_t code_bytes(const Rows &t) { return (size_t)t.n * t.chunks * 4; }
size_t scale_count(const Rows &t) { return (size_t)t.n * t.groups; }

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return cz::set_error(CZ_E_HIP, "%s: %s", what, hipGetErrorString(e));
    return CZ_OK;
}

// the product kernel's launch: digits of the queries, workgroups that stay while their waves go over the table
struct ProductPlan {
    uint32_t steps, ct, grid_x, grid_y, n_tiles, lds;
    u32x4 *digits;
    int *exponent;
    float *qnorm;
};
ProductPlan product_plan(const Rows &t, uint32_t B, bool near, cz::Carve &c) {
    ProductPlan p;
    p.steps = (t.groups << t.gshift) / 64 + ((t.groups << t.gshift) % 64 != 0);
    p.n_tiles = (uint32_t)(((uint64_t)t.n + kTile - 1) / kTile);
    const uint32_t blocks4 = (B + 3) / 4;
    p.ct = blocks4 >= 4 && p.steps * 4 <= 64 ? 4 : blocks4 >= 2 && p.steps * 2 <= 64 ? 2 : 1;
    p.lds = p.ct * p.steps * 1024;
    p.grid_y = (blocks4 + p.ct - 1) / p.ct;
    const uint32_t per_cu = std::max(1u, std::min((uint32_t)residents((int)p.ct, (int)t.gshift), 160u * 1024 / p.lds));
    p.grid_x = std::max(1u, std::min((p.n_tiles + 3) / 4, std::max(1u, 256 * per_cu / p.grid_y)));
    p.digits = c.take<u32x4>((size_t)blocks4 * p.steps * 64);
    p.exponent = c.take<int>(B);
    p.qnorm = near ? c.take<float>(B) : nullptr;
    return p;
}

// c of score_error for the digit products.  With |.| the 2-norm and x the row as it stands: the fixed point moves an element by at most
// 2^-31 of the largest, 2^-31 |q| sqrt(dim) |x| in all; joining the digits and adding `groups` terms rounds by 2^-24 of sums that
// |q| |x| bounds (three times it, as digits of both signs may cancel); the cosine's reciprocal root, its product and the norm's own
// rounding are below 2^-21.  A hundredth on top for the bound's own arithmetic.
float score_error_unit(const Rows &t) {
    return 1.01f * (3.f * (float)(t.groups + 4) * 0x1p-24f + sqrtf((float)t.dim) * 0x1p-31f + 0x1p-21f);
}

template <int CT, int GS, bool SW, bool NEAR>
int launch_product_as(const Rows &t, const ProductPlan &p, uint32_t B, float *out, const Near &near, hipStream_t stream) {
    auto kernel = q4_product_kernel<CT, GS, SW, NEAR>;
    if (p.lds > 65536) CZ_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds));
    hipLaunchKernelGGL(kernel, dim3(p.grid_x, p.grid_y), dim3(256), p.lds, stream, t, p.digits, p.exponent, B, p.steps, out, near);
    return CZ_OK;
}
template <int CT, int GS, bool NEAR>
int launch_product_gs(const Rows &t, const ProductPlan &p, uint32_t B, float *out, const Near &near, hipStream_t stream) {
    // whole batches of scales, each row's aligned to the load: rows of whole 128-byte lines of codes
    const bool sw = t.chunks % 32 == 0 && (reinterpret_cast<uintptr_t>(t.scales) & 15) == 0;
    return sw ? launch_product_as<CT, GS, true, NEAR>(t, p, B, out, near, stream) : launch_product_as<CT, GS, false, NEAR>(t, p, B, out, near, stream);
}
template <int CT, bool NEAR>
int launch_product_ct(const Rows &t, const ProductPlan &p, uint32_t B, float *out, const Near &near, hipStream_t stream) {
    if (t.gshift == 5) return launch_product_gs<CT, 5, NEAR>(t, p, B, out, near, stream);
    if (t.gshift == 6) return launch_product_gs<CT, 6, NEAR>(t, p, B, out, near, stream);
    return launch_product_gs<CT, 7, NEAR>(t, p, B, out, near, stream);
}
template <bool NEAR>
int launch_product(const Rows &t, const ProductPlan &p, const float *q, uint32_t B, float *out, const Near &near, hipStream_t stream) {
    const uint32_t fixed = p.steps * 1024;  // the four queries' fixed point
    if (fixed > 65536) CZ_HIP(hipFuncSetAttribute((const void *)q4_digits_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)fixed));
    hipLaunchKernelGGL(q4_digits_kernel, dim3((B + 3) / 4), dim3(256), fixed, stream, q, B, t.dim, p.steps, (uint32_t *)p.digits, p.exponent, p.qnorm);
    if (p.ct == 4) return launch_product_ct<4, NEAR>(t, p, B, out, near, stream);
    if (p.ct == 2) return launch_product_ct<2, NEAR>(t, p, B, out, near, stream);
    return launch_product_ct<1, NEAR>(t, p, B, out, near, stream);
}

// Saved work (queries x rows x dim) from which scores come first.  Some k of the tiles stay to be looked at.  The f64 distances of all rows run at some 2e12 elements a second, the scores' launches
// take 30 us whatever they do; 644 x 18221 x 312: 1928 us without scores, 180 with them (k = 11, 285
// tiles); 569 x 11596 x 584, k = 51, 182 tiles: 1489 and 516
constexpr double kFilterFrom = 6e7;
// Up to so many queries the digits' product (100 us for each 16 of them at 1M x 768) is the faster way to the scores; at 48 both take 0.37 ms.
constexpr uint32_t kDigitQueries = 32;
using Tile128 = gemm::Tile<gemm::F16, 128, 128, 2, 2>;
using Tile256 = gemm::Tile<gemm::F16, 256, 256, 2, 4>;

// c of score_error for the f16 product (derived at its kernel); the cosine's own rounding and the bound's as for the digits
float half_error_unit(const Rows &t) {
    return 1.01f * (0x1p-11f + sqrtf((float)t.dim) * 0x1p-20f + (float)t.dim * 0x1p-24f + 0x1p-21f);
}

// queries of one launch; a larger batch goes in turns through the same scratch: 1 GiB of tile scores, twice that where the f16 product turns them, for
// tables of up to 268M rows; beyond, what 64 queries take (8.6 GB, and as much again, at 2^31 rows)
uint32_t turn_of(const Rows &t) {
    const uint64_t n_tiles = std::max<uint64_t>(1, ((uint64_t)t.n + kTile - 1) / kTile);
    return (uint32_t)std::min<uint64_t>(4096, std::max<uint64_t>(64, (1ull << 28) / n_tiles));
}

struct KnnPlan {
    uint32_t chunks, tiles_per_chunk;
    bool filtered;         // scores first, f64 distances of the tiles that can hold a result only
    uint64_t *part_key;
    uint32_t *part_id, *part_count;
    ProductPlan product;
    int halves;            // scores by the f16 product: 0 no, 1 with 128 x 128 tiles, 2 with 256 x 256
    uint32_t steps, parts, ldb;
    _Float16 *q16;
    int *exponent;
    float *turned;
    float *qnorm, *tile_score, *tile_norm, *best, *need;
    double *limit;
    uint32_t n_best;
    size_t bytes;
};
KnnPlan knn_plan(const Rows &t, uint32_t B, uint32_t k, void *ws) {
    KnnPlan p{};
    const uint32_t n_tiles = (uint32_t)(((uint64_t)t.n + kTile - 1) / kTile);
    p.filtered = n_tiles > k && (double)B * t.n * t.dim * (n_tiles - k) / n_tiles >= kFilterFrom;
    // enough workgroups to fill the chip, few enough lists to join
    uint32_t chunks = std::min(n_tiles, std::max(1u, (p.filtered ? 512 : 2048) / B));
    if (p.filtered && B > 256) chunks = 2;
    chunks = std::max(1u, std::min(chunks, std::max(16u, 65536 / k)));
    p.tiles_per_chunk = std::max(1u, (n_tiles + chunks - 1) / chunks);
    p.chunks = std::max(1u, (n_tiles + p.tiles_per_chunk - 1) / p.tiles_per_chunk);
    cz::Carve c(ws);
    p.part_key = c.take<uint64_t>((size_t)B * p.chunks * k);
    p.part_id = c.take<uint32_t>((size_t)B * p.chunks * k);
    p.part_count = c.take<uint32_t>((size_t)B * p.chunks);
    if (p.filtered) {
        p.steps = (t.groups << t.gshift) / 64 + ((t.groups << t.gshift) % 64 != 0);
        // 256 queries to a tile, unless 128 leave fewer columns unused (384 queries against 1M x 768: 0.93 ms instead of 1.10; 1024: 2.44 and 2.26)
        p.halves = B <= kDigitQueries ? 0 : (B + 127) / 128 * 128 < (B + 255) / 256 * 256 ? 1 : 2;
        if (p.halves) {
            const uint32_t b = p.halves == 2 ? 256 : 128, qt = (B + b - 1) / b, blocks = (t.n + b - 1) / b, resident = p.halves == 2 ? 256 : 512;
            p.parts = std::max(1u, std::min(blocks, resident / qt));
            p.n_best = p.parts * 2;
            p.ldb = (B + 31) / 32 * 32;
            p.q16 = c.take<_Float16>((size_t)B * p.steps * 64);
            p.exponent = c.take<int>(B);
            p.qnorm = c.take<float>(B);
            p.turned = c.take<float>((size_t)n_tiles * p.ldb);
        } else {
            p.product = product_plan(t, B, true, c);
            p.n_best = p.product.grid_x * 4;
            p.qnorm = p.product.qnorm;
        }
        p.tile_score = c.take<float>((size_t)B * n_tiles);
        p.tile_norm = c.take<float>(n_tiles);
        p.best = c.take<float>((size_t)B * p.n_best);
        p.need = c.take<float>(B);
        p.limit = c.take<double>(B);
    }
    p.bytes = c.used();
    return p;
}

template <class G>
int launch_scores(const Rows &t, const KnnPlan &p, uint32_t B, const Near &near, hipStream_t stream) {
    const gemm::Operand Q{(const char *)p.q16, (uint64_t)p.steps * 128, B};
    const uint32_t blocks = (uint32_t)(((uint64_t)t.n + G::BM - 1) / G::BM), lds = G::kLds + G::BM * 8, qt = (B + G::BN - 1) / G::BN;
    auto kernel = t.gshift == 5 ? q4_scores_kernel<G, 5> : t.gshift == 6 ? q4_scores_kernel<G, 6> : q4_scores_kernel<G, 7>;
    CZ_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, dim3(p.parts * qt), dim3(G::kThreads), lds, stream, t, Q, p.exponent, p.steps, near, p.turned, p.ldb, blocks,
                       (blocks + p.parts - 1) / p.parts);
    return CZ_OK;
}
// the scores of every tile, what rows are sure to reach: by digits or in f16
int launch_near(const Rows &t, const KnnPlan &p, const float *q, uint32_t B, const Near &near, hipStream_t stream) {
    if (!p.halves) return launch_product<true>(t, p.product, q, B, nullptr, near, stream);
    hipLaunchKernelGGL(q4_halves_kernel, dim3((B + 3) / 4), dim3(256), 0, stream, q, B, t.dim, p.steps, p.q16, p.exponent, p.qnorm);
    hipLaunchKernelGGL(q4_tile_norm_kernel, dim3((near.n_tiles + 3) / 4), dim3(256), 0, stream, near.sqnorms, t.n, p.tile_norm);
    const int rc = p.halves == 2 ? launch_scores<Tile256>(t, p, B, near, stream) : launch_scores<Tile128>(t, p, B, near, stream);
    if (rc) return rc;
    hipLaunchKernelGGL(q4_turn_kernel, dim3((near.n_tiles + 63) / 64, (B + 63) / 64), dim3(256), 0, stream, p.turned, near.n_tiles, B, p.ldb, p.tile_score);
    return CZ_OK;
}

int check_codes(const uint8_t *codes, const uint16_t *scales) {
    if (!codes || !scales) return cz::set_error(CZ_E_INVALID, "null table");
    return CZ_OK;
}
int check_codes_device(const uint8_t *codes, const uint16_t *scales) {
    if (reinterpret_cast<uintptr_t>(codes) & 15) return cz::set_error(CZ_E_INVALID, "codes are not 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(scales) & 1) return cz::set_error(CZ_E_INVALID, "scales are not aligned");
    int rc = cz::check_device_ptr(codes, "codes");
    return rc ? rc : cz::check_device_ptr(scales, "scales");
}

}  // namespace

extern "C" int cz_q4_quantize(const void *vectors, int elem, uint32_t n, uint32_t dim, uint64_t ld, uint32_t group, uint8_t *codes,
                              uint16_t *scales, float *sqnorms, uint32_t flags, void *stream_) {
    Rows t;
    int rc = shape_of_rows(n, dim, group, &t);
    if (rc) return rc;
    if (elem != CZ_ELEM_F32 && elem != CZ_ELEM_BF16) return cz::set_error(CZ_E_INVALID, "unknown element type %d", elem);
    if (ld < dim) return cz::set_error(CZ_E_INVALID, "ld is smaller than dim");
    rc = cz::ensure_device();
    if (rc) return rc;
    if (n == 0) return CZ_OK;
    if (!vectors || !sqnorms) return cz::set_error(CZ_E_INVALID, "null buffer");
    rc = check_codes(codes, scales);
    if (rc) return rc;
    hipStream_t stream = (hipStream_t)stream_;
    cz::HostStage stage(stream);
    const bool dev = flags & CZ_DEVICE_PTRS;
    const size_t es = elem == CZ_ELEM_F32 ? 4 : 2;
    const uint8_t *x = (const uint8_t *)vectors;
    if (dev) {
        if ((rc = check_codes_device(codes, scales)) || (rc = cz::check_device_ptr(vectors, "vectors")) ||
            (rc = cz::check_device_ptr(sqnorms, "sqnorms")))
            return rc;
        if ((reinterpret_cast<uintptr_t>(vectors) % es) || (reinterpret_cast<uintptr_t>(sqnorms) & 3))
            return cz::set_error(CZ_E_INVALID, "vectors or sqnorms are not aligned to their elements");
    } else {
        if ((rc = stage.in((const uint8_t *)vectors, ((size_t)(n - 1) * ld + dim) * es, &x)) ||
            (rc = stage.out(codes, code_bytes(t), &codes)) || (rc = stage.out(scales, scale_count(t), &scales)) ||
            (rc = stage.out(sqnorms, (size_t)n, &sqnorms)))
            return rc;
    }
    const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ld * es) % 16 == 0;
    const uint32_t lpr = std::max(lanes_per_row(t.chunks), group / 8);
    const uint32_t grid = std::min((n + 256 / lpr - 1) / (256 / lpr), 1u << 22);  // (a launch has fewer than 2^32 threads)
#define CZ_Q4_CALL(L)                                                                                                              \
    if (elem == CZ_ELEM_F32)                                                                                                       \
        hipLaunchKernelGGL((q4_quantize_kernel<float, L>), dim3(grid), dim3(256), 0, stream, (const float *)x, ld, wide, t, codes, \
                           scales, sqnorms);                                                                                       \
    else                                                                                                                           \
        hipLaunchKernelGGL((q4_quantize_kernel<uint16_t, L>), dim3(grid), dim3(256), 0, stream, (const uint16_t *)x, ld, wide, t,  \
                           codes, scales, sqnorms)
    CZ_Q4_LANES(lpr, CZ_Q4_CALL);
#undef CZ_Q4_CALL
    rc = launched("cz_q4_quantize");
    if (rc || dev) return rc;
    return stage.finish();
}

extern "C" int cz_q4_dequantize(const uint8_t *codes, const uint16_t *scales, uint32_t n, uint32_t dim, uint32_t group,
                                const uint32_t *rows, uint32_t m, float *out, uint32_t flags, void *stream_) {
    Rows t;
    int rc = shape_of_rows(n, dim, group, &t);
    if (rc) return rc;
    if (!rows && m != n) return cz::set_error(CZ_E_INVALID, "without row numbers all n rows are decoded: m must be n");
    rc = cz::ensure_device();
    if (rc) return rc;
    if (m == 0) return CZ_OK;
    if (!out) return cz::set_error(CZ_E_INVALID, "null buffer");
    if (n) {
        rc = check_codes(codes, scales);
        if (rc) return rc;
    }
    hipStream_t stream = (hipStream_t)stream_;
    cz::HostStage stage(stream);
    const bool dev = flags & CZ_DEVICE_PTRS;
    if (dev) {
        if ((rc = check_codes_device(codes, scales)) || (rc = cz::check_device_ptr(rows, "rows")) || (rc = cz::check_device_ptr(out, "out")))
            return rc;
        if ((reinterpret_cast<uintptr_t>(rows) & 3) || (reinterpret_cast<uintptr_t>(out) & 3))
            return cz::set_error(CZ_E_INVALID, "rows or out are not aligned to their elements");
    } else {
        if (rows)
            for (uint32_t i = 0; i < m; i++)
                if (rows[i] >= n) return cz::set_error(CZ_E_INVALID, "rows[%u] = %u is no row of %u", i, rows[i], n);
        if ((rc = stage.in(codes, code_bytes(t), &codes)) || (rc = stage.in(scales, scale_count(t), &scales)) ||
            (rows && (rc = stage.in(rows, m, &rows))) || (rc = stage.out(out, (size_t)m * dim, &out)))
            return rc;
    }
    t.codes = codes;
    t.scales = scales;
    const bool wide = dim % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const uint64_t blocks = std::min<uint64_t>(((uint64_t)m * t.chunks + 255) / 256, 1u << 20);
    hipLaunchKernelGGL(q4_dequantize_kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, t, rows, m, wide, out);
    rc = launched("cz_q4_dequantize");
    if (rc || dev) return rc;
    return stage.finish();
}

extern "C" uint64_t cz_q4_workspace(uint32_t n, uint32_t dim, uint32_t group, uint32_t B, uint32_t k) {
    Rows t;
    if (shape_of_rows(n, dim, group, &t) || k > 1024) return 0;
    if (B == 0 || n == 0) return 256;
    const uint32_t turn = turn_of(t);
    // the last turn of a large batch is smaller and may be laid out differently
    size_t need = 0;
    for (const uint32_t nb : {std::min(B, turn), B > turn && B % turn ? B % turn : 0u}) {
        if (!nb) continue;
        cz::Carve c(nullptr);
        if (k == 0) (void)product_plan(t, nb, false, c);
        need = std::max(need, k ? knn_plan(t, nb, k, nullptr).bytes : c.used());
    }
    return need;
}

extern "C" int cz_q4_dots(const uint8_t *codes, const uint16_t *scales, uint32_t n, uint32_t dim, uint32_t group,
                          const float *queries, uint32_t B, float *out, void *ws, uint64_t ws_bytes, uint32_t flags, void *stream_) {
    Rows t;
    int rc = shape_of_rows(n, dim, group, &t);
    if (rc) return rc;
    rc = cz::ensure_device();
    if (rc) return rc;
    if (n == 0 || B == 0) return CZ_OK;
    if (!queries || !out) return cz::set_error(CZ_E_INVALID, "null buffer");
    rc = check_codes(codes, scales);
    if (rc) return rc;
    hipStream_t stream = (hipStream_t)stream_;
    cz::HostStage stage(stream);
    cz::DevBuf<uint8_t> own;
    const bool dev = flags & CZ_DEVICE_PTRS;
    if (dev) {
        if ((rc = check_codes_device(codes, scales)) || (rc = cz::check_device_ptr(queries, "queries")) || (rc = cz::check_device_ptr(out, "out")))
            return rc;
        if ((reinterpret_cast<uintptr_t>(queries) & 3) || (reinterpret_cast<uintptr_t>(out) & 3))
            return cz::set_error(CZ_E_INVALID, "queries or out are not aligned to their elements");
    } else {
        if ((rc = stage.in(codes, code_bytes(t), &codes)) || (rc = stage.in(scales, scale_count(t), &scales)) ||
            (rc = stage.in(queries, (size_t)B * dim, &queries)) || (rc = stage.out(out, (size_t)B * n, &out)))
            return rc;
        ws = nullptr;
    }
    void *base = nullptr;
    if ((rc = cz::scratch_of(ws, ws_bytes, cz_q4_workspace(n, dim, group, B, 0), own, &base))) return rc;
    t.codes = codes;
    t.scales = scales;
    const uint32_t turn = turn_of(t);
    for (uint32_t b0 = 0; b0 < B; b0 += turn) {
        const uint32_t nb = std::min(turn, B - b0);
        cz::Carve c(base);
        const ProductPlan p = product_plan(t, nb, false, c);
        if ((rc = launch_product<false>(t, p, queries + (size_t)b0 * dim, nb, out + (size_t)b0 * n, Near{}, stream))) return rc;
    }
    rc = launched("cz_q4_dots");
    if (rc) return rc;
    if (!dev) return stage.finish();
    if (own.p) CZ_HIP(hipStreamSynchronize(stream));
    return CZ_OK;
}

extern "C" int cz_q4_knn(int metric, const uint8_t *codes, const uint16_t *scales, const float *sqnorms, uint32_t n, uint32_t dim,
                         uint32_t group, const float *queries, uint32_t B, uint32_t k, int has_radius, double radius,
                         uint32_t *out_ids, double *out_dist, uint32_t *out_count, void *ws, uint64_t ws_bytes,
                         const volatile uint8_t *poison, uint32_t flags, void *stream_) {
    Rows t;
    int rc = shape_of_rows(n, dim, group, &t);
    if (rc) return rc;
    if (metric != CZ_L2 && metric != CZ_COSINE && metric != CZ_IP) return cz::set_error(CZ_E_INVALID, "unknown metric %d", metric);
    if (k == 0 || k > 1024) return cz::set_error(CZ_E_UNSUPPORTED, "k must be in 1..1024");
    rc = cz::ensure_device();
    if (rc) return rc;
    if (B == 0) return CZ_OK;
    if (!queries || !out_ids || !out_dist || !out_count) return cz::set_error(CZ_E_INVALID, "null buffer");
    if (n) {
        rc = check_codes(codes, scales);
        if (rc) return rc;
        if (!sqnorms) return cz::set_error(CZ_E_INVALID, "null buffer");
    }
    if (cz::poisoned(poison)) return cz::set_error(CZ_E_CANCELLED, "cancelled");
    hipStream_t stream = (hipStream_t)stream_;
    cz::HostStage stage(stream);
    cz::DevBuf<uint8_t> own;
    const bool dev = flags & CZ_DEVICE_PTRS;
    if (dev) {
        if ((rc = check_codes_device(codes, scales)) || (rc = cz::check_device_ptr(sqnorms, "sqnorms")) ||
            (rc = cz::check_device_ptr(queries, "queries")) || (rc = cz::check_device_ptr(out_ids, "out_ids")) ||
            (rc = cz::check_device_ptr(out_dist, "out_dist")) || (rc = cz::check_device_ptr(out_count, "out_count")))
            return rc;
        if ((reinterpret_cast<uintptr_t>(queries) & 3) || (reinterpret_cast<uintptr_t>(sqnorms) & 3) || (reinterpret_cast<uintptr_t>(out_ids) & 3) ||
            (reinterpret_cast<uintptr_t>(out_dist) & 7) || (reinterpret_cast<uintptr_t>(out_count) & 3))
            return cz::set_error(CZ_E_INVALID, "an array is not aligned to its elements");
    } else {
        if ((rc = stage.in(codes, code_bytes(t), &codes)) || (rc = stage.in(scales, scale_count(t), &scales)) ||
            (rc = stage.in(sqnorms, (size_t)n, &sqnorms)) || (rc = stage.in(queries, (size_t)B * dim, &queries)) ||
            (rc = stage.out(out_ids, (size_t)B * k, &out_ids)) || (rc = stage.out(out_dist, (size_t)B * k, &out_dist)) ||
            (rc = stage.out(out_count, (size_t)B, &out_count)))
            return rc;
        ws = nullptr;
    }
    void *base = nullptr;
    if ((rc = cz::scratch_of(ws, ws_bytes, cz_q4_workspace(n, dim, group, B, k), own, &base))) return rc;
    t.codes = codes;
    t.scales = scales;
    const size_t smem = 256 * 12 + 1024 * 4 + (size_t)k * 12 + 64 + (size_t)t.chunks * 64;
    const uint32_t lpr = lanes_per_row(t.chunks);
    const uint32_t turn = turn_of(t);
    for (uint32_t b0 = 0; b0 < B; b0 += turn) {
        const uint32_t nb = std::min(turn, B - b0);
        const float *q = queries + (size_t)b0 * dim;
        KnnPlan p{};
        if (n) {
            p = knn_plan(t, nb, k, base);
            Candidates cand{};
            if (p.filtered) {
                const float err = p.halves ? half_error_unit(t) : score_error_unit(t);
                const Near near{metric, sqnorms, err, p.qnorm, p.tile_score, p.tile_norm, p.best, (n + kTile - 1) / kTile, p.n_best};
                if ((rc = launch_near(t, p, q, nb, near, stream))) return rc;
                hipLaunchKernelGGL(q4_need_kernel, dim3(nb), dim3(1024), 0, stream, near, p.n_best < 4 * k, k, p.need, p.limit);
                cand = Candidates{p.tile_score, p.tile_norm, p.qnorm, p.need, p.limit, err};
            }
#define CZ_Q4_CALL(L)                                                                                                              \
    hipLaunchKernelGGL((q4_scan_kernel<L>), dim3(p.chunks, nb), dim3(256), smem, stream, metric, t, q, k, p.tiles_per_chunk, cand, \
                       p.part_key, p.part_id, p.part_count)
#define CZ_Q4_ALLOW(L) CZ_HIP(hipFuncSetAttribute((const void *)q4_scan_kernel<L>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem))
            if (smem > 65536) CZ_Q4_LANES(lpr, CZ_Q4_ALLOW);
            CZ_Q4_LANES(lpr, CZ_Q4_CALL);
#undef CZ_Q4_CALL
#undef CZ_Q4_ALLOW
        }
        hipLaunchKernelGGL(q4_join_kernel, dim3(nb), dim3(256), join_lds(k), stream, p.part_key, p.part_id,
                           p.part_count, p.chunks, k,
                           has_radius, radius, out_ids + (size_t)b0 * k, out_dist + (size_t)b0 * k, out_count + b0);
    }
    rc = launched("cz_q4_knn");
    if (rc) return rc;
    if (!dev) return stage.finish();
    if (own.p) CZ_HIP(hipStreamSynchronize(stream));
    return CZ_OK;
}
