// softmax_xent.hip -- softmax cross entropy over a whole table and its gradient (arithmetic: include/cozo_gpu.h).
//
// Forward: one matrix product per (table tile, query tile) with the softmax's running maximum and sum as its epilogue.  The TABLE rows are
// the product's m and the queries its n: a lane's accumulators then belong to one query, so maximum and sum run in the lane and lanes are
// joined once, at the end of a workgroup's stretch of the table.  Stretches are joined in a second launch.
// Gradient, a piece of the table at a time:  P = grad_loss scale (softmax - onehot) of the piece is computed again and stored (in f32 in both
// orders, in bf16 once: the matrix loop then reads P, Q and W turned where k is not what is contiguous), then  dW = P^T Q  is written and
// dq += P W  goes to per-stretch partial sums (each added to by one workgroup only, in a fixed order: no atomics).
// A bf16 P takes one product for each gradient where a P in two parts would take two (some 4.5 ms on top of 7.8 for 1024 x 1M x 768): rows of dW
// that answer nothing are off by 0.0020 to 0.0024 of their size (rounding the result alone: 0.0017).  What it rounds off matters most at the
// answers -- the largest entries, which may well carry all the same value and so the same error -- and is kept there in f32, its term added to
// dW's row and to dq.  In f32 the answer's entry is left out of dq's long sum, which would lose the small terms beside it, and added at its end.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "call.h"
#include "gemm_nt.h"

using gemm::Bf16;
using gemm::F32;
using gemm::Operand;
using gemm::Ragged;
using gemm::Tailed;
using gemm::Turned;

namespace {

constexpr uint32_t kMaxDim = 8192;
uint32_t tiles_of(uint64_t n, uint32_t b) { return (uint32_t)((n + b - 1) / b); }
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__bf16 x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T down(float x) { return (T)x; }
__device__ __forceinline__ bool has_answer(uint32_t y, uint32_t V) { return y < V; }
// what exponents are taken relative to: a maximum of -inf (nothing seen yet, or nothing but -inf) or +inf is no reference
__device__ __forceinline__ float reference(float m) { return fabsf(m) < __builtin_inff() ? m : 0.f; }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// place of element (row, k) of a matrix of `rows` rows in panels of k (gemm_nt.h)
template <typename T>
__device__ __forceinline__ uint64_t in_panels(uint32_t row, uint32_t k, uint32_t rows) {
    constexpr uint32_t W = 128 / sizeof(T);
    return ((uint64_t)(k / W) * rows + row) * W + k % W;
}

// rows of x, their first dim elements and zeros up to ldo, one 16-byte aligned row behind the other, and rows of zeros up to `rows`; with targets
// given also for those whose target is no row of the table (as in xent_transpose_kernel)
template <typename T>
__global__ void __launch_bounds__(256)
xent_pack_kernel(const T *__restrict__ x, uint64_t ld, uint32_t n, uint32_t dim, T *__restrict__ out, uint32_t ldo, uint32_t rows,
                 const uint32_t *__restrict__ targets, uint32_t V) {
    const uint64_t total = (uint64_t)rows * ldo;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / ldo), c = (uint32_t)(i - (uint64_t)r * ldo);
        out[i] = c < dim && r < n && (!targets || has_answer(targets[r], V)) ? x[r * ld + c] : (T)0.f;
    }
}

// out[d][r] = x[r][d] in panels of r, for d < dim, r < n, and zeros up to r = width; rows whose target is no row of the table are zeros too
// when targets are given (what such a query holds, NaN included, must not reach a product with its zero weight).  HBM bound: 64 x 64 through
// LDS, 16 bytes of a row read and written at a time.  `wide`: rows of x are 16-byte aligned.  width is a multiple of a panel's.
template <typename T>
__global__ void __launch_bounds__(256)
xent_transpose_kernel(const T *__restrict__ x, uint64_t ld, bool wide, uint32_t n, uint32_t dim, const uint32_t *__restrict__ targets, uint32_t V,
                      T *__restrict__ out, uint32_t width) {
    constexpr int P = 16 / sizeof(T);  // elements of 16 bytes
    typedef T Piece __attribute__((ext_vector_type(P)));
    __shared__ T tile[64][64 + 4 / sizeof(T)];
    const uint32_t r0 = blockIdx.x * 64, d0 = blockIdx.y * 64;
#pragma unroll
    for (uint32_t i = 0; i < 16 / P; i++) {
        const uint32_t at = i * 256 + threadIdx.x, row = at / (64 / P), c = at % (64 / P) * P, r = r0 + row, d = d0 + c;
        Piece v;
#pragma unroll
        for (int j = 0; j < P; j++) v[j] = (T)0.f;
        if (r < n && (!targets || has_answer(targets[r], V))) {
            const T *src = x + r * ld + d;
            if (wide && d + P <= dim) v = *(const Piece *)src;
            else
#pragma unroll
                for (int j = 0; j < P; j++)
                    if (d + j < dim) v[j] = src[j];
        }
#pragma unroll
        for (int j = 0; j < P; j++) tile[row][c + j] = v[j];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 16 / P; i++) {
        const uint32_t at = i * 256 + threadIdx.x, row = at / (64 / P), c = at % (64 / P) * P, d = d0 + row, r = r0 + c;
        if (d >= dim || r >= width) continue;
        Piece v;
#pragma unroll
        for (int j = 0; j < P; j++) v[j] = tile[c + j][row];
        *(Piece *)(out + in_panels<T>(d, r, dim)) = v;
    }
}

// scale log2(e) in two parts: a factor rounded to f32 would move all logits alike.  low has high's sign and is not zero where high is not, so that
// infinite products stay what they are; the least f32 there is moves a finite product by less than 1e-6.  (|scale| < 2^127: in the f32 range)
struct Scale2 {
    float high, low;
    static Scale2 of(float scale) {
        const double x = (double)scale * 1.44269504088896340736;
        if (x == 0.0) return Scale2{0.f, 0.f};
        float high = (float)x;
        if (std::fabs((double)high) > std::fabs(x)) high = std::nextafter(high, 0.f);
        return Scale2{high, std::copysign(std::max((float)std::fabs(x - (double)high), 0x1p-149f), high)};
    }
};

// From here on neighbouring f32 logits are 1 and more apart: what a product's rounding leaves of a difference can be any number.
constexpr float kCoarse = 16777216.f;

// l relative to reference m, a whole number or infinite, made relative to ref
template <typename T>
__device__ __forceinline__ T moved(T l, float m, float ref) {
    if (m == -__builtin_inff()) return l;
    const int by = (int)fminf(fmaxf(m - ref, -1100.f), 1100.f);
    if constexpr (sizeof(T) == 8) return ldexp(l, by);
    else return ldexpf(l, by);
}

// A tile's products taken into the running reference m and sum l of each of the lane's queries, to base 2.  The reference is the largest product (the
// least one where the scale is negative), scaled once, and from there the next whole number, so that a sum moves from one reference to another
// without being rounded, however often a table's rows beat the ones before them.  A term is then two fused multiply-adds, an exponential and an addition,
// and no product is rounded before the difference.  A tile's terms are added in four f32 sums, tiles in f64: a single f32 sum over a stretch lost
// more with every row (33000 queries, 1M rows: lse off by 9e-4; the time of both is the same).  PART: only the first `left` rows exist.
template <class G, bool PART>
__device__ __forceinline__ void take(const G &g, uint32_t left, Scale2 scale2, float (&m)[G::NT], double (&l)[G::NT]) {
    const int lane = threadIdx.x & 63;
    const bool least = scale2.high < 0.f;
    const float none = least ? __builtin_inff() : -__builtin_inff();
    auto is_there = [&](int i, int r) { return (uint32_t)(G::wave_row() + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) < left; };
#pragma unroll
    for (int j = 0; j < G::NT; j++) {
        float top = none;
        if (__builtin_expect(least, 0)) {
#pragma unroll
            for (int i = 0; i < G::MT; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = fminf(top, !PART || is_there(i, r) ? g.acc[i][j][r] : none);
        } else {
#pragma unroll
            for (int i = 0; i < G::MT; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, !PART || is_there(i, r) ? g.acc[i][j][r] : none);
        }
        top = ceilf(fmaxf(m[j], top * scale2.high));
        const float ref = reference(top);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        if (__builtin_expect(!__any(!(fabsf(ref) < kCoarse)), 1)) {
#pragma unroll
            for (int i = 0; i < G::MT; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float e = exp2_(fmaf(g.acc[i][j][r], scale2.low, fmaf(g.acc[i][j][r], scale2.high, -ref)));
                    sum[r & 3] += !PART || is_there(i, r) ? e : 0.f;
                }
        } else {  // (whole numbers: the largest term is to be 1)
#pragma unroll
            for (int i = 0; i < G::MT; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float e = exp2_(__fsub_rn(__fmul_rn(g.acc[i][j][r], scale2.high), ref));
                    sum[r & 3] += !PART || is_there(i, r) ? e : 0.f;
                }
        }
        l[j] = moved(l[j], m[j], ref) + (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
        m[j] = top;
    }
}

template <class G, class O>
__global__ void __launch_bounds__(G::kThreads)
xent_forward_kernel(O W, Operand Q, uint32_t steps, Scale2 scale2, uint32_t n_tiles, uint32_t tiles_per_part,
                    float2 *__restrict__ parts) {
    constexpr int BM = G::BM, BN = G::BN, WM = G::WM, WN = G::WN;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t qt = (Q.rows + BN - 1) / BN, at = gemm::place_in_order();
    const uint32_t n0 = at % qt * BN, part = at / qt;
    const uint32_t t0 = part * tiles_per_part, t1 = min(n_tiles, t0 + tiles_per_part);
    float m[G::NT];
    double l[G::NT];
#pragma unroll
    for (int j = 0; j < G::NT; j++) m[j] = -__builtin_inff(), l[j] = 0.0;
    G g;
    for (uint32_t t = t0; t < t1; t++) {
        g.run(W, t * BM, Q, n0, 0, steps, lds);
        const uint32_t left = W.rows - t * BM;  // rows of this tile that exist
        if (__builtin_expect(left >= BM, 1)) take<G, false>(g, left, scale2, m, l);
        else take<G, true>(g, left, scale2, m, l);
        __syncthreads();  // LDS is free for the next tile
    }
    // lanes that hold the same query: the two halves, then the waves along m
    float2 *red = (float2 *)lds;  // [WM][BN]
#pragma unroll
    for (int j = 0; j < G::NT; j++) {
        const float mo = __shfl_xor(m[j], 32, 64);
        const double lo = __shfl_xor(l[j], 32, 64);
        const float top = fmaxf(m[j], mo), ref = reference(top);
        const float sum = (float)(moved(l[j], m[j], ref) + moved(lo, mo, ref));
        if (lane < 32) red[(threadIdx.x >> 6) / WN * BN + G::wave_col() + j * 32 + lane] = make_float2(top, sum);
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < BN; c += G::kThreads) {
        if (n0 + c >= Q.rows) break;
        float2 a = red[c];
#pragma unroll
        for (int w = 1; w < WM; w++) {
            const float2 b = red[w * BN + c];
            const float top = fmaxf(a.x, b.x), ref = reference(top);
            a.y = moved(a.y, a.x, ref) + moved(b.y, b.x, ref);
            a.x = top;
        }
        parts[(uint64_t)part * Q.rows + n0 + c] = a;
    }
}

// one wave per query: the stretches joined, the answer's logit, the loss.  f64: a handful of operations per query
template <typename T>
__global__ void __launch_bounds__(256)
xent_join_kernel(const float2 *__restrict__ parts, uint32_t n_parts, const T *__restrict__ q, uint64_t ldq, const T *__restrict__ w,
                 uint64_t ldw, uint32_t Tn, uint32_t V, uint32_t dim, const uint32_t *__restrict__ targets, float scale,
                 float *__restrict__ loss, float *__restrict__ lse) {
    const uint32_t t = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (t >= Tn) return;
    float top = -__builtin_inff();
    for (uint32_t p = lane; p < n_parts; p += 64) top = fmaxf(top, parts[(uint64_t)p * Tn + t].x);
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float ref = reference(top);
    double sum = 0.0;
    for (uint32_t p = lane; p < n_parts; p += 64) {
        const float2 a = parts[(uint64_t)p * Tn + t];
        sum += a.x == -__builtin_inff() ? (double)a.y : (double)a.y * exp2((double)a.x - (double)ref);
    }
    const uint32_t y = targets[t];
    double z = 0.0;
    if (has_answer(y, V))
        for (uint32_t d = lane; d < dim; d += 64) z = fma((double)up(q[t * ldq + d]), (double)up(w[y * ldw + d]), z);
    for (int o = 32; o; o >>= 1) {
        sum += __shfl_xor(sum, o, 64);
        z += __shfl_xor(z, o, 64);
    }
    if (lane) return;
    const double e = ((double)ref + log2(sum)) * 0.69314718055994530942;
    lse[t] = (float)e;
    loss[t] = y == CZ_NONE ? 0.f : y < V ? (float)(e - (double)scale * z) : __builtin_nanf("");
}

// P of a piece: p[t][v] and pt[v][t], in panels of v and of t, zeros where the piece or the queries (up to tp) end; rest[t]: what rounding
// the answer's entry cut off (bf16), or that entry, which p then has as 0 (f32)
template <class G, class O>
__global__ void __launch_bounds__(G::kThreads)
xent_weights_kernel(O W, uint32_t v0, uint32_t V, Operand Q, uint32_t steps, float scale, const uint32_t *__restrict__ targets,
                    const float *__restrict__ lse, const float *__restrict__ grad_loss, typename G::Elem::T *__restrict__ p,
                    typename G::Elem::T *__restrict__ pt, uint32_t vp, uint32_t tp, float *__restrict__ rest) {
    typedef typename G::Elem E;
    constexpr int BM = G::BM, BN = G::BN;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t qt = (tp + BN - 1) / BN;
    const uint32_t at = gemm::place_in_order(), n0 = at % qt * BN, m0 = at / qt * BM;
    const int lane = threadIdx.x & 63;
    G g;
    g.run(W, m0, Q, n0, 0, steps, lds);
    constexpr bool kSplit = sizeof(typename E::T) == 2;
#pragma unroll
    for (int j = 0; j < G::NT; j++) {
        const uint32_t t = n0 + G::wave_col() + j * 32 + (lane & 31);
        const uint32_t y = t < Q.rows ? targets[t] : CZ_NONE;
        const bool on = t < Q.rows && has_answer(y, V);
        const float e = on ? lse[t] : 0.f, weight = on ? grad_loss[t] * scale : 0.f;
        const float most = fabsf(e) < kCoarse ? __builtin_inff() : 0.f;  // of z - lse (NaN stays)
#pragma unroll
        for (int i = 0; i < G::MT; i++)
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                const uint32_t v = m0 + G::wave_row() + i * 32 + 8 * r4 + 4 * (lane >> 5);
                typename E::T o[4], own[4];  // for dW and for dq
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    // (to base 2 only after the difference: log2(e) lse and log2(e) scale, rounded, would be an error that a query's entries share)
                    const float below = fmaf(g.acc[i][j][4 * r4 + r], scale, -e);
                    float x = exp2_((below > most ? most : below) * kLog2e);
                    const bool hit = on && v0 + v + r == y;
                    if (hit) x -= 1.f;
                    x = on && v + r < W.rows ? x * weight : 0.f;
                    o[r] = down<typename E::T>(x);
                    if (hit) rest[t] = kSplit ? x - up(o[r]) : x;
                    own[r] = !kSplit && hit ? (typename E::T)0.f : o[r];
                }
                if (t < tp && p) {
                    typedef typename E::T T4 __attribute__((ext_vector_type(4)));
                    *(T4 *)(p + in_panels<typename E::T>(t, v, tp)) = T4{own[0], own[1], own[2], own[3]};
                }
                if (t < tp && pt)
#pragma unroll
                    for (int r = 0; r < 4; r++) pt[in_panels<typename E::T>(v + r, t, vp)] = o[r];
            }
    }
}

// what is left of the answers' own terms
template <typename T>
struct Answers {
    const uint32_t *targets;
    const float *rest;
    const T *q, *w;
    uint64_t ldq, ldw;
    uint32_t T_n, V;
};

// grad_table rows of a piece (rows v0 ... of the table): pt . qt^T, and the rest for the queries that the rows answer
template <class G, class O>
__global__ void __launch_bounds__(G::kThreads)
xent_table_grad_kernel(O Pt, O Qt, uint32_t steps, Answers<typename G::Elem::T> an, uint32_t v0, uint32_t rows,
                       typename G::Elem::T *__restrict__ out, uint32_t dim) {
    constexpr int BM = G::BM, BN = G::BN, kWaves = G::kThreads / 64;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t nt = (dim + BN - 1) / BN;
    const uint32_t at = gemm::place_in_order(), n0 = at % nt * BN, m0 = at / nt * BM;
    G g;
    g.run(Pt, m0, Qt, n0, 0, steps, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t *count = (uint32_t *)lds, *list = count + kWaves;  // of each wave; the queries that rows of this tile answer, ascending
    if (sizeof(typename G::Elem::T) == 2 && an.rest)
    for (uint32_t t0 = 0; t0 < an.T_n; t0 += G::kThreads) {
        const uint32_t t = t0 + threadIdx.x, y = t < an.T_n ? an.targets[t] : CZ_NONE;
        const bool here = y < an.V && y >= v0 + m0 && y - v0 - m0 < BM;
        if (!__syncthreads_or(here)) continue;  // (the LDS is free after it: the product's last reads lie before)
        const unsigned long long m = __ballot(here);
        if (lane == 0) count[wave] = __popcll(m);
        __syncthreads();
        uint32_t first = 0, total = 0;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            if (w < wave) first += count[w];
            total += count[w];
        }
        if (here) list[first + __popcll(m & ((1ull << lane) - 1ull))] = t;
        __syncthreads();
        for (uint32_t i = 0; i < total; i++) {
            const uint32_t tq = list[i];
            const int row = (int)(an.targets[tq] - v0 - m0) - G::wave_row() - 4 * (lane >> 5);
            if (row < -4 || row >= BM / G::WM) continue;  // (another wave's)
            const float rest = an.rest[tq];
#pragma unroll
            for (int j = 0; j < G::NT; j++) {
                const uint32_t c = n0 + G::wave_col() + j * 32 + (lane & 31);
                const float x = c < dim ? up(an.q[tq * an.ldq + c]) * rest : 0.f;
#pragma unroll
                for (int k = 0; k < G::MT; k++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (row == k * 32 + 8 * (r >> 2) + (r & 3)) g.acc[k][j][r] += x;
            }
        }
        __syncthreads();
    }
    g.each([&](uint32_t r, uint32_t c, float v) {
        if (m0 + r < rows && n0 + c < dim) out[(uint64_t)(m0 + r) * dim + n0 + c] = down<typename G::Elem::T>(v);
    });
}

// partial sums of grad_queries: part s gets p . wt^T over the steps of stretch s, added to what the earlier pieces left there
template <class G, class O>
__global__ void __launch_bounds__(G::kThreads)
xent_query_grad_kernel(Operand P, O Wt, uint32_t T, uint32_t steps, uint32_t steps_per_part, int add, float *__restrict__ parts, uint32_t dim) {
    constexpr int BM = G::BM, BN = G::BN;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t nt = (dim + BN - 1) / BN, mt = (T + BM - 1) / BM;
    const uint32_t at = gemm::place_in_order(), n0 = at % nt * BN, m0 = at / nt % mt * BM, s = at / (nt * mt);
    const uint32_t s0 = s * steps_per_part, s1 = min(steps, s0 + steps_per_part);
    float *out = parts + (uint64_t)s * T * dim;
    G g;
    if (s0 < s1) g.run(P, m0, Wt, n0, s0, s1 - s0, lds);
    else g.zero();
    g.each([&](uint32_t r, uint32_t c, float v) {
        if (m0 + r < T && n0 + c < dim) {
            float *o = out + (uint64_t)(m0 + r) * dim + n0 + c;
            *o = add ? *o + v : v;
        }
    });
}

// grad_queries: the partial sums added up, and the rest for the rows that answer; four lanes to an element, 16 loads on their way in each
// (255 queries, 96 wide, 256 sums: 8 us; with four loads 32)
template <typename T>
__global__ void __launch_bounds__(256)
xent_sum_parts_kernel(const float *__restrict__ parts, uint32_t n_parts, uint64_t n, uint32_t dim, Answers<T> an, T *__restrict__ out) {
    __shared__ float sums[4][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint64_t i0 = (uint64_t)blockIdx.x * 64; i0 < n; i0 += (uint64_t)gridDim.x * 64) {
        const uint64_t i = i0 + lane;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        if (i < n) {
            uint32_t p = wave;
            for (; p + 4 * 15 < n_parts; p += 64) {  // (16 loads on their way)
                float v[16];
#pragma unroll
                for (int u = 0; u < 16; u++) v[u] = parts[(p + 4 * u) * n + i];
#pragma unroll
                for (int u = 0; u < 16; u++) a[u & 3] += v[u];
            }
            for (; p < n_parts; p += 4) a[0] += parts[p * n + i];
        }
        sums[wave][lane] = (a[0] + a[1]) + (a[2] + a[3]);
        __syncthreads();
        if (wave == 0 && i < n) {
            float v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
            if (an.targets) {
                const uint32_t t = (uint32_t)(i / dim), y = an.targets[t];
                // (without an answer: zero weights, which a table row that is not finite would have made more of)
                v = has_answer(y, an.V) ? v + an.rest[t] * up(an.w[y * an.ldw + (i - (uint64_t)t * dim)]) : 0.f;
            }
            out[i] = down<T>(v);
        }
        __syncthreads();
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
uint64_t up_to(uint64_t x, uint64_t m) { return (x + m - 1) / m * m; }

struct Shape {
    uint32_t T, V, dim;
    uint64_t ldq, ldw;
    bool bf16;
    uint32_t es() const { return bf16 ? 2 : 4; }
    uint32_t kstep() const { return 128 / es(); }
    uint32_t kp() const { return (uint32_t)up_to(dim, kstep()); }
    uint32_t tp() const { return (uint32_t)up_to(T, kstep()); }
};

struct Plan {
    uint32_t piece;        // backward: table rows worked on at a time
    uint32_t parts;        // forward: stretches of the table; backward: partial sums of grad_queries
    int fwd, of_p, of_w, of_q;  // tiles (TileOf): forward's; backward's of P, of grad_table, of grad_queries
    void *q, *w;           // packed copies: of queries that are unaligned or no whole steps wide; of a piece of an unaligned bf16 table (gradient)
    void *qt, *wt, *p, *pt;  // (bf16: qt is a copy of the queries without those that have no answer, wt and pt are not needed)
    float2 *stats;
    float *dq, *rest;
    size_t bytes;
};

// Tiles of the four products, table rows (or, for grad_queries, queries) first.  Large: most products for what is read; the smaller ones where
// large tiles would leave CUs without work; narrow and flat for a few queries, which do not spend the matrix cores on columns that are not there
// (4 queries, 17601 rows of 840 in f32: 277 us with 128 x 128 throughout, 148 with these).
template <class E> using Large = gemm::Tile<E, 256, 256, 2, 4>;
template <class E> using Small = gemm::Tile<E, 128, 128, 2, 2>;
template <class E> using Tiny = gemm::Tile<E, 64, 64, 2, 2>;
template <class E> using Narrow = gemm::Tile<E, 128, 32, 4, 1>;
template <class E> using Flat = gemm::Tile<E, 32, 128, 1, 4>;
// (in f32 the products over rows and queries have no large tile: see large_in_f32)
template <class E> using Long = std::conditional_t<sizeof(typename E::T) == 2, Large<E>, Small<E>>;
enum TileOf { kLarge, kSmall, kTiny, kNarrow, kFlat };
constexpr uint32_t kFull = 192;  // tiles (one to a CU) that are taken to fill the chip's 256 CUs

uint32_t rows_of(TileOf t) { return t == kLarge ? 256 : t == kTiny ? 64 : t == kFlat ? 32 : 128; }
uint32_t cols_of(TileOf t) { return t == kLarge ? 256 : t == kTiny ? 64 : t == kNarrow ? 32 : 128; }
uint64_t count_of(TileOf t, uint64_t m, uint64_t n) { return (m + rows_of(t) - 1) / rows_of(t) * ((n + cols_of(t) - 1) / cols_of(t)); }
// the largest tile with which m x n fills the chip
TileOf filling(bool large, uint64_t m, uint64_t n) {
    if (large && m > 128 && n > 128 && count_of(kLarge, m, n) >= kFull) return kLarge;
    return count_of(kSmall, m, n) >= kFull ? kSmall : kTiny;
}

// f32's matrix instructions take 16 times as long for what is read, so that large tiles are no gain, and with 128 accumulators a lane has no room
// for more than one sum; but over few steps what a tile costs besides them counts (small and large tiles, 255 queries x 100003 rows, 96 wide:
// forward 76 and 65 us, weights 100 and 93; loss + gradient of 645 x 32103, 165 wide: 471 and 488)
bool large_in_f32(uint32_t dim) { return dim <= 128; }

// f of the tile that t says; LARGE, TINY and OTHER: what a product has under these names
template <class E, class LARGE, class TINY, class OTHER, class F>
int with_tile(int t, F f) {
    return t == kLarge ? f(LARGE{}) : t == kSmall ? f(Small<E>{}) : t == kTiny ? f(TINY{}) : f(OTHER{});
}

// rows that the matrix loop can read where they are (the queries also need whole steps: theirs are the zeros behind a row)
bool direct(const void *x, uint64_t ld, uint32_t dim, uint32_t es) {
    return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * es % 16 == 0 && dim * es % 16 == 0;
}

Plan make_plan(const Shape &s, bool grad, void *ws) {
    // the scratch asked for covers packed copies whether or not a call needs them: alignment is not known here
    // (a piece is 256 MiB of the wider of P's and the table's rows, but at least 1024 rows: past 65536 queries in f32, 131072 in bf16, P grows with
    // them, by 8 KiB (both orders) and 2 KiB for each)
    Plan pl{};
    const uint64_t es = s.es(), kp = s.kp(), tp = s.tp();
    const uint64_t budget = 256ull << 20;
    const uint64_t per_row = es * (grad ? std::max<uint64_t>(tp, kp) : kp);
    pl.piece = (uint32_t)std::min<uint64_t>(up_to(s.V, 256), std::max<uint64_t>(1024, budget / per_row / 1024 * 1024));
    cz::Carve c(ws);
    pl.q = c.take<uint8_t>((uint64_t)s.T * kp * es);
    if (!grad) {
        pl.fwd = s.T <= 32 ? kNarrow : filling(s.bf16 || large_in_f32(s.dim), s.V, s.T);
        const TileOf f = (TileOf)pl.fwd;
        const uint32_t qt = tiles_of(s.T, cols_of(f)), tiles = tiles_of(s.V, rows_of(f));
        const uint32_t resident = f == kLarge ? 256 : f == kSmall ? 512 : 1024;
        pl.parts = std::max(1u, std::min(tiles, resident / qt));
        pl.stats = c.take<float2>((uint64_t)pl.parts * s.T);
    } else {
        pl.qt = c.take<uint8_t>(kp * tp * es);
        pl.p = c.take<uint8_t>(tp * pl.piece * es);
        if (s.bf16) pl.w = c.take<uint8_t>((uint64_t)pl.piece * kp * es);
        if (!s.bf16) {
            pl.wt = c.take<uint8_t>((uint64_t)s.dim * pl.piece * es);
            pl.pt = c.take<uint8_t>(pl.piece * tp * es);
        }
        const uint32_t nv = std::min(s.V, pl.piece);
        const uint32_t steps = (uint32_t)up_to(nv, 256) / s.kstep(), most = std::max(1u, steps / 8);  // stretches of at least 8 steps
        pl.of_p = s.T <= 32 ? kNarrow : filling(s.bf16 || large_in_f32(s.dim), nv, tp);
        pl.of_w = filling(s.bf16, nv, s.dim);
        pl.of_q = s.T <= 32 ? kFlat : s.bf16 && s.T > 128 && s.dim > 128 && count_of(kLarge, s.T, s.dim) * most >= kFull ? kLarge : kSmall;
        const uint32_t tiles = (uint32_t)count_of((TileOf)pl.of_q, s.T, s.dim), resident = pl.of_q == kLarge ? 256 : pl.of_q == kSmall ? 512 : 1024;
        pl.parts = std::max(1u, std::min({resident / tiles, most, 256u}));
        pl.rest = c.take<float>(s.T);
        pl.dq = c.take<float>((uint64_t)pl.parts * s.T * s.dim);
    }
    pl.bytes = c.used();
    return pl;
}

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return cz::set_error(CZ_E_HIP, "%s: %s", what, hipGetErrorString(e));
    return CZ_OK;
}
uint32_t grid_of(uint64_t items) { return (uint32_t)std::min<uint64_t>((items + 255) / 256, 1u << 16); }

template <typename T>
void pack(const T *x, uint64_t ld, uint32_t n, uint32_t dim, void *out, uint32_t ldo, hipStream_t stream, uint32_t rows = 0,
          const uint32_t *targets = nullptr, uint32_t V = 0) {
    rows = std::max(n, rows);
    hipLaunchKernelGGL(xent_pack_kernel<T>, dim3(grid_of((uint64_t)rows * ldo)), dim3(256), 0, stream, x, ld, n, dim, (T *)out, ldo, rows, targets, V);
}

// a kernel over tiles G, with the LDS that they ask for
template <class G, class K, class... A>
int launch(K kernel, uint32_t grid, hipStream_t stream, A... args) {
    if (G::kLds > 65536) CZ_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, G::kLds));
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(G::kThreads), G::kLds, stream, args...);
    return CZ_OK;
}
// f over W's rows of dim elements where they are: as they are, with zeros behind rows that end inside a step, or element by element aligned
template <typename T, class F>
int over(const Operand &W, uint32_t dim, bool aligned, F f) {
    const uint32_t bytes = dim * sizeof(T);
    if (!aligned) return f(Ragged<T>{W, W.rows, bytes});
    return bytes % 128 ? f(Tailed{W, W.rows, bytes}) : f(W);
}
template <class G, class O>
int forward_over(const O &W, const Operand &Q, uint32_t steps, Scale2 scale2, uint32_t parts, float2 *stats, hipStream_t stream) {
    const uint32_t tiles = tiles_of(W.rows, G::BM);
    return launch<G>(xent_forward_kernel<G, O>, parts * tiles_of(Q.rows, G::BN), stream, W, Q, steps, scale2, tiles, (tiles + parts - 1) / parts, stats);
}

template <class E>
int forward(const Shape &s, const Plan &pl, const void *q_, const void *w_, const uint32_t *targets, float scale, float *loss, float *lse,
            hipStream_t stream) {
    typedef typename E::T T;
    const T *q = (const T *)q_, *w = (const T *)w_;
    const uint32_t es = s.es(), kp = s.kp(), steps = kp / s.kstep();
    Operand Q{(const char *)q, s.ldq * es, s.T};
    if (!direct(q, s.ldq, s.dim, es) || s.dim != kp) {
        pack(q, s.ldq, s.T, s.dim, pl.q, kp, stream);
        Q = Operand{(const char *)pl.q, (uint64_t)kp * es, s.T};
    }
    const Operand W{(const char *)w, s.ldw * es, s.V};
    const int rc = over<T>(W, s.dim, direct(w, s.ldw, s.dim, es), [&](const auto &O) {
        auto go = [&](auto g) { return forward_over<decltype(g)>(O, Q, steps, Scale2::of(scale), pl.parts, pl.stats, stream); };
        return with_tile<E, Large<E>, Tiny<E>, Narrow<E>>(pl.fwd, go);
    });
    if (rc) return rc;
    hipLaunchKernelGGL(xent_join_kernel<T>, dim3((s.T + 3) / 4), dim3(256), 0, stream, pl.stats, pl.parts, q, s.ldq, w, s.ldw, s.T, s.V, s.dim,
                       targets, scale, loss, lse);
    return launched("cz_softmax_xent");
}

template <typename T>
void transpose(const T *x, uint64_t ld, uint32_t n, uint32_t dim, const uint32_t *targets, uint32_t V, void *out, uint32_t width, hipStream_t stream) {
    const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * sizeof(T) % 16 == 0;
    hipLaunchKernelGGL(xent_transpose_kernel<T>, dim3((width + 63) / 64, (dim + 63) / 64), dim3(256), 0, stream, x, ld, wide, n, dim, targets, V,
                       (T *)out, width);
}

template <class G, class O>
int weights_of(const O &W, uint32_t v0, uint32_t V, const Operand &Q, uint32_t steps, float scale, const uint32_t *targets, const float *lse,
               const float *grad_loss, void *p, uint32_t vp, void *pt, uint32_t tp, float *rest, hipStream_t stream) {
    typedef typename G::Elem::T T;
    return launch<G>(xent_weights_kernel<G, O>, tiles_of(vp, G::BM) * tiles_of(tp, G::BN), stream, W, v0, V, Q, steps, scale, targets, lse, grad_loss,
                     (T *)p, (T *)pt, vp, tp, rest);
}
template <class G, class O>
int table_grad_of(const O &Pt, const O &Qt, uint32_t steps, const Answers<typename G::Elem::T> &an, uint32_t v0,
                  uint32_t rows, typename G::Elem::T *out, uint32_t dim, hipStream_t stream) {
    return launch<G>(xent_table_grad_kernel<G, O>, tiles_of(rows, G::BM) * tiles_of(dim, G::BN), stream, Pt, Qt, steps, an, v0, rows, out, dim);
}
template <class G, class O>
int query_grad_of(const Operand &P, const O &Wt, uint32_t T, uint32_t steps, uint32_t parts, bool add, float *dq, uint32_t dim, hipStream_t stream) {
    return launch<G>(xent_query_grad_kernel<G, O>, tiles_of(T, G::BM) * tiles_of(dim, G::BN) * parts, stream, P, Wt, T, steps,
                     (steps + parts - 1) / parts, add ? 1 : 0, dq, dim);
}

template <class E>
int backward(const Shape &s, const Plan &pl, const void *q_, const void *w_, const uint32_t *targets, float scale, const float *lse,
             const float *grad_loss, void *dq, void *dw, hipStream_t stream) {
    typedef typename E::T T;
    const T *q = (const T *)q_, *w = (const T *)w_;
    const uint32_t es = s.es(), kp = s.kp(), tp = s.tp(), steps = kp / s.kstep();
    Operand Q{(const char *)q, s.ldq * es, s.T};
    if (!direct(q, s.ldq, s.dim, es) || s.dim != kp) {
        pack(q, s.ldq, s.T, s.dim, pl.q, kp, stream);
        Q = Operand{(const char *)pl.q, (uint64_t)kp * es, s.T};
    }
    const bool wd = direct(w, s.ldw, s.dim, es);
    const Answers<T> an{targets, pl.rest, q, w, s.ldq, s.ldw, s.T, s.V};
    constexpr bool kTurned = sizeof(T) == 2;  // (there is no transposing read for f32)
    if (dw) {
        if (kTurned) pack(q, s.ldq, s.T, s.dim, pl.qt, kp, stream, tp, targets, s.V);
        else transpose(q, s.ldq, s.T, s.dim, targets, s.V, pl.qt, tp, stream);
    }
    for (uint32_t v0 = 0; v0 < s.V; v0 += pl.piece) {
        const uint32_t nv = std::min(pl.piece, s.V - v0), vp = (uint32_t)up_to(nv, 256);
        const T *wv = w + v0 * s.ldw;
        Operand W{(const char *)wv, s.ldw * es, nv};
        const bool packed = kTurned && !wd;  // (to be read turned, rows of 8 have to be aligned)
        if (packed) {
            pack(wv, s.ldw, nv, s.dim, pl.w, kp, stream);
            W = Operand{(const char *)pl.w, (uint64_t)kp * es, nv};
        }
        void *p = dq || kTurned ? pl.p : nullptr, *pt = dw && !kTurned ? pl.pt : nullptr;
        int rc = over<T>(W, packed ? kp : s.dim, wd || packed, [&](const auto &O) {
            auto go = [&](auto g) { return weights_of<decltype(g)>(O, v0, s.V, Q, steps, scale, targets, lse, grad_loss, p, vp, pt, tp, pl.rest, stream); };
            return with_tile<E, Large<E>, Tiny<E>, Narrow<E>>(pl.of_p, go);
        });
        if (rc) return rc;
        const uint32_t vsteps = vp / s.kstep();
        if (dq) {
            const Operand P = gemm::panels(pl.p, tp);
            auto query_grad = [&](const auto &Wt) {
                auto go = [&](auto g) { return query_grad_of<decltype(g)>(P, Wt, s.T, vsteps, pl.parts, v0 != 0, pl.dq, s.dim, stream); };
                return with_tile<E, Long<E>, Flat<E>, Flat<E>>(pl.of_q, go);
            };
            if constexpr (kTurned) {
                rc = query_grad(Turned{W.base, W.ld, 128, wd ? s.dim : kp, nv});
            } else {
                transpose(wv, s.ldw, nv, s.dim, (const uint32_t *)nullptr, 0u, pl.wt, vp, stream);
                rc = query_grad(gemm::panels(pl.wt, s.dim));
            }
            if (rc) return rc;
        }
        if (dw) {
            T *out = (T *)dw + (uint64_t)v0 * s.dim;
            auto table_grad = [&](const auto &Pt, const auto &Qt) {
                auto go = [&](auto g) { return table_grad_of<decltype(g)>(Pt, Qt, tp / s.kstep(), an, v0, nv, out, s.dim, stream); };
                return with_tile<E, Long<E>, Tiny<E>, Tiny<E>>(pl.of_w, go);
            };
            if constexpr (kTurned) rc = table_grad(Turned{(const char *)pl.p, 128, tp * 128ull, vp, tp}, Turned{(const char *)pl.qt, (uint64_t)kp * es, 128, kp, tp});
            else rc = table_grad(gemm::panels(pl.pt, vp), gemm::panels(pl.qt, s.dim));
            if (rc) return rc;
        }
    }
    if (dq)
        hipLaunchKernelGGL(xent_sum_parts_kernel<T>, dim3(grid_of((uint64_t)s.T * s.dim * 4)), dim3(256), 0, stream, pl.dq, pl.parts,
                           (uint64_t)s.T * s.dim, s.dim, an, (T *)dq);
    return launched("cz_softmax_xent_grad");
}

int check_shape(uint32_t T, uint32_t V, uint32_t dim, int elem) {
    if (elem != CZ_ELEM_F32 && elem != CZ_ELEM_BF16) return cz::set_error(CZ_E_INVALID, "unknown element type %d", elem);
    if (dim == 0 || dim > kMaxDim) return cz::set_error(CZ_E_UNSUPPORTED, "dim must be in 1..%u", kMaxDim);
    if (V == 0) return cz::set_error(CZ_E_INVALID, "a softmax over no rows");
    if (V >= 0x80000000u || T >= (1u << 24)) return cz::set_error(CZ_E_UNSUPPORTED, "fewer than 2^31 rows and 2^24 queries");
    return CZ_OK;
}

// what forward and backward check alike; host arrays are staged
int prepare_call(Shape &s, int elem, float scale, uint32_t flags, const void *&queries, const void *&table, const uint32_t *&targets,
                 cz::HostStage &stage) {
    int rc = check_shape(s.T, s.V, s.dim, elem);
    if (rc) return rc;
    if (!(std::fabs(scale) < 0x1p127f)) return cz::set_error(CZ_E_INVALID, "scale is not below 2^127");
    s.bf16 = elem == CZ_ELEM_BF16;
    if (s.ldq < s.dim || s.ldw < s.dim) return cz::set_error(CZ_E_INVALID, "ldq or ldw is smaller than dim");
    rc = cz::ensure_device();
    if (rc || s.T == 0) return rc;
    if (!queries || !table || !targets) return cz::set_error(CZ_E_INVALID, "null buffer");
    const uint32_t es = s.es();
    if (flags & CZ_DEVICE_PTRS) {
        if ((reinterpret_cast<uintptr_t>(queries) | reinterpret_cast<uintptr_t>(table)) % es || reinterpret_cast<uintptr_t>(targets) % 4)
            return cz::set_error(CZ_E_INVALID, "an array is not aligned to its elements");
        if ((rc = cz::check_device_ptr(queries, "queries")) || (rc = cz::check_device_ptr(table, "table"))) return rc;
        return cz::check_device_ptr(targets, "targets");
    }
    for (uint32_t t = 0; t < s.T; t++)
        if (targets[t] != CZ_NONE && targets[t] >= s.V) return cz::set_error(CZ_E_INVALID, "targets[%u] = %u is no row of %u", t, targets[t], s.V);
    const uint8_t *q = (const uint8_t *)queries, *w = (const uint8_t *)table;
    if ((rc = stage.in(q, ((uint64_t)(s.T - 1) * s.ldq + s.dim) * es, &q)) || (rc = stage.in(w, ((uint64_t)(s.V - 1) * s.ldw + s.dim) * es, &w)) ||
        (rc = stage.in(targets, s.T, &targets)))
        return rc;
    queries = q;
    table = w;
    return CZ_OK;
}

}  // namespace

extern "C" uint64_t cz_softmax_xent_workspace(uint32_t T, uint32_t V, uint32_t dim, int elem, int grad) {
    if (check_shape(T, V, dim, elem)) return 0;
    if (T == 0) return 256;
    return make_plan(Shape{T, V, dim, dim, dim, elem == CZ_ELEM_BF16}, grad != 0, nullptr).bytes;
}

extern "C" int cz_softmax_xent(const void *queries, uint64_t ldq, const void *table, uint64_t ldw, int elem, uint32_t T, uint32_t V,
                               uint32_t dim, const uint32_t *targets, float scale, float *loss, float *lse, void *ws, uint64_t ws_bytes,
                               uint32_t flags, void *stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    cz::HostStage stage(stream);
    cz::DevBuf<uint8_t> own;
    Shape s{T, V, dim, ldq, ldw, false};
    int rc = prepare_call(s, elem, scale, flags, queries, table, targets, stage);
    if (rc || T == 0) return rc;
    if (!loss || !lse) return cz::set_error(CZ_E_INVALID, "null buffer");
    const bool dev = flags & CZ_DEVICE_PTRS;
    if (dev) {
        if ((reinterpret_cast<uintptr_t>(loss) | reinterpret_cast<uintptr_t>(lse)) & 3)
            return cz::set_error(CZ_E_INVALID, "an array is not aligned to its elements");
        if ((rc = cz::check_device_ptr(loss, "loss")) || (rc = cz::check_device_ptr(lse, "lse"))) return rc;
    } else {
        if ((rc = stage.out(loss, T, &loss)) || (rc = stage.out(lse, T, &lse))) return rc;
        ws = nullptr;
    }
    void *base = nullptr;
    if ((rc = cz::scratch_of(ws, ws_bytes, make_plan(s, false, nullptr).bytes, own, &base))) return rc;
    const Plan pl = make_plan(s, false, base);
    rc = s.bf16 ? forward<Bf16>(s, pl, queries, table, targets, scale, loss, lse, stream)
                : forward<F32>(s, pl, queries, table, targets, scale, loss, lse, stream);
    if (rc) return rc;
    if (!dev) return stage.finish();
    if (own.p) CZ_HIP(hipStreamSynchronize(stream));
    return CZ_OK;
}

extern "C" int cz_softmax_xent_grad(const void *queries, uint64_t ldq, const void *table, uint64_t ldw, int elem, uint32_t T, uint32_t V,
                                    uint32_t dim, const uint32_t *targets, float scale, const float *lse, const float *grad_loss,
                                    void *grad_queries, void *grad_table, void *ws, uint64_t ws_bytes, uint32_t flags, void *stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    cz::HostStage stage(stream);
    cz::DevBuf<uint8_t> own;
    Shape s{T, V, dim, ldq, ldw, false};
    const bool dev = flags & CZ_DEVICE_PTRS;
    int rc = prepare_call(s, elem, scale, flags, queries, table, targets, stage);
    if (rc || (!grad_queries && !grad_table)) return rc;
    const uint32_t es = s.es();
    if (T == 0) {  // the table's gradient is written whole all the same
        if (!grad_table) return CZ_OK;
        if (!dev) {
            std::fill_n((uint8_t *)grad_table, (size_t)V * dim * es, (uint8_t)0);
            return CZ_OK;
        }
        if ((rc = cz::check_device_ptr(grad_table, "grad_table"))) return rc;
        if (s.bf16)
            hipLaunchKernelGGL(xent_sum_parts_kernel<__bf16>, dim3(grid_of((uint64_t)V * dim * 4)), dim3(256), 0, stream, (const float *)nullptr, 0u,
                               (uint64_t)V * dim, dim, Answers<__bf16>{}, (__bf16 *)grad_table);
        else
            hipLaunchKernelGGL(xent_sum_parts_kernel<float>, dim3(grid_of((uint64_t)V * dim * 4)), dim3(256), 0, stream, (const float *)nullptr, 0u,
                               (uint64_t)V * dim, dim, Answers<float>{}, (float *)grad_table);
        return launched("cz_softmax_xent_grad");
    }
    if (!lse || !grad_loss) return cz::set_error(CZ_E_INVALID, "null buffer");
    if (dev) {
        if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(grad_loss)) & 3 ||
            (reinterpret_cast<uintptr_t>(grad_queries) | reinterpret_cast<uintptr_t>(grad_table)) % es)
            return cz::set_error(CZ_E_INVALID, "an array is not aligned to its elements");
        if ((rc = cz::check_device_ptr(lse, "lse")) || (rc = cz::check_device_ptr(grad_loss, "grad_loss")) ||
            (rc = cz::check_device_ptr(grad_queries, "grad_queries")) || (rc = cz::check_device_ptr(grad_table, "grad_table")))
            return rc;
    } else {
        uint8_t *dq = (uint8_t *)grad_queries, *dw = (uint8_t *)grad_table;
        if ((rc = stage.in(lse, T, &lse)) || (rc = stage.in(grad_loss, T, &grad_loss)) ||
            (dq && (rc = stage.out(dq, (size_t)T * dim * es, &dq))) || (dw && (rc = stage.out(dw, (size_t)V * dim * es, &dw))))
            return rc;
        grad_queries = dq;
        grad_table = dw;
        ws = nullptr;
    }
    void *base = nullptr;
    if ((rc = cz::scratch_of(ws, ws_bytes, make_plan(s, true, nullptr).bytes, own, &base))) return rc;
    const Plan pl = make_plan(s, true, base);
    rc = s.bf16 ? backward<Bf16>(s, pl, queries, table, targets, scale, lse, grad_loss, grad_queries, grad_table, stream)
                : backward<F32>(s, pl, queries, table, targets, scale, lse, grad_loss, grad_queries, grad_table, stream);
    if (rc) return rc;
    if (!dev) return stage.finish();
    if (own.p) CZ_HIP(hipStreamSynchronize(stream));
    return CZ_OK;
}
