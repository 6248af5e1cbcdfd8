// q4.hip -- 4-bit rows with group scales: quantising, decoding, products with queries, exhaustive k-NN (form and arithmetic:
// include/cozo_gpu.h).
#include <algorithm>
#include <cmath>

#include "call.h"
#include "distance.h"
#include "topk.h"

using namespace czd;

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kMaxDim = 8192;
constexpr uint32_t kMaxBatch = 4096;  // queries of one launch; a larger batch goes in turns through the same scratch

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
    const uint64_t r = (uint64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int glanes = 1 << (t.gshift - 3);
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

// ---- products, the simple form: LPR lanes per row, every query in turn ------------------------------------------------
template <int LPR>
__global__ void __launch_bounds__(256)
q4_dots_kernel(Rows t, const float *__restrict__ q, uint32_t B, float *__restrict__ out) {
    const int sub = threadIdx.x % LPR;
    const uint64_t r = (uint64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    if (r >= t.n) return;
    for (uint32_t b = 0; b < B; b++) {
        float a = 0.f;
        for (uint32_t c = sub; c < t.chunks; c += LPR) {
            const uint32_t w = *(const uint32_t *)(t.codes + (r * t.chunks + c) * 4);
            const float s = bf16_to_f32(t.scales[r * t.groups + ((c * 8) >> t.gshift)]);
            float p = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c * 8 + j < t.dim) {
                    const float qv = q[(uint64_t)b * t.dim + c * 8 + j];
                    p = fma_((float)code_at(w, j), fabsf(qv) < __builtin_inff() ? qv : __builtin_nanf(""), p);
                }
            a = fma_(p, s, a);
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) a += __shfl_xor(a, o, 64);
        if (sub == 0) out[(uint64_t)b * t.n + r] = a;
    }
}

// ---- exact k-NN ------------------------------------------------------------------------------------------------------
// the f64 distance of one row from the query in LDS, by LPR neighbouring lanes (every lane returns it).  Codes times scales and the
// products with an f32 are exact in f64; the lanes' sums are joined by a fixed butterfly, so equal rows have equal bits.
template <int LPR>
__device__ __forceinline__ double row_distance(int metric, const Rows &t, uint32_t r, int sub, const float *q, double qq) {
    double a = 0.0, x2 = 0.0;
    for (uint32_t c = sub; c < t.chunks; c += LPR) {
        const uint32_t w = *(const uint32_t *)(t.codes + ((uint64_t)r * t.chunks + c) * 4);
        const double s = (double)bf16_to_f32(t.scales[(uint64_t)r * t.groups + ((c * 8) >> t.gshift)]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (c * 8 + j >= t.dim) break;
            const double x = (double)code_at(w, j) * s, qv = (double)q[c * 8 + j];
            if (metric == CZ_L2) {
                const double d = qv - x;
                a = fma(d, d, a);
            } else {
                a = fma(qv, x, a);
                x2 = fma(x, x, x2);
            }
        }
    }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) {
        a += __shfl_xor(a, o, 64);
        x2 += __shfl_xor(x2, o, 64);
    }
    if (metric == CZ_L2) return a;
    if (metric == CZ_COSINE) return 1.0 - a / sqrt(qq * x2);
    return 1.0 - a;
}

constexpr uint32_t kTile = 64;  // rows that are looked at together

// per (chunk of tiles, query): the k nearest rows of the chunk as a sorted partial list
template <int LPR>
__global__ void __launch_bounds__(256)
q4_scan_kernel(int metric, Rows t, const float *__restrict__ queries, uint32_t k, uint32_t tiles_per_chunk,
               uint64_t *__restrict__ part_key, uint32_t *__restrict__ part_id) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    uint64_t *bkey = (uint64_t *)smem_raw;       // [256]
    uint64_t *tkey = bkey + 256;                  // [k]
    double *red = (double *)(tkey + k);           // [4]
    uint32_t *bid = (uint32_t *)(red + 4);        // [256]
    uint32_t *tid_ = bid + 256;                   // [k]
    float *q = (float *)(tid_ + k);               // [dim]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = tid % LPR;
    const uint32_t b = blockIdx.y;
    const uint64_t n_tiles = (t.n + kTile - 1) / kTile;
    double qq = 0.0;
    for (uint32_t i = tid; i < t.dim; i += 256) {
        const float v = queries[(uint64_t)b * t.dim + i];
        q[i] = v;
        qq = fma((double)v, (double)v, qq);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) qq += __shfl_xor(qq, o, 64);
    if (lane == 0) red[wave] = qq;
    __syncthreads();
    qq = (red[0] + red[1]) + (red[2] + red[3]);
    const uint64_t t0 = (uint64_t)blockIdx.x * tiles_per_chunk, t1 = min(n_tiles, t0 + tiles_per_chunk);
    int tcnt = 0;
    for (uint64_t r0 = t0 * kTile; r0 < t1 * kTile; r0 += 256) {
        const uint32_t nb = (uint32_t)min((uint64_t)256, min((uint64_t)t.n, t1 * kTile) - r0);
        for (int it = 0; it < LPR; it++) {
            const uint32_t slot = wave * 64 + it * (64 / LPR) + lane / LPR;
            if (wave * 64 + it * (64 / LPR) >= (int)nb) break;  // (uniform in the wave)
            const uint32_t r = (uint32_t)(r0 + min(slot, nb - 1));
            const double d = row_distance<LPR>(metric, t, r, sub, q, qq);
            if (sub == 0 && slot < nb) {
                bkey[slot] = dist_key(d);
                bid[slot] = r;
            }
        }
        tcnt = topk_merge_batch((int)nb, bkey, bid, tkey, tid_, tcnt, (int)k);
    }
    const size_t o = ((size_t)b * gridDim.x + blockIdx.x) * k;
    for (uint32_t i = tid; i < k; i += 256) {
        const bool have = (int)i < tcnt;
        part_key[o + i] = have ? tkey[i] : ~0ull;
        part_id[o + i] = have ? tid_[i] : CZ_NONE;
    }
}

// one workgroup per query: the partial lists joined, the radius cut, the padding
__global__ void __launch_bounds__(256)
q4_join_kernel(const uint64_t *__restrict__ part_key, const uint32_t *__restrict__ part_id, uint32_t n_parts, uint32_t k,
               int has_radius, double radius, uint32_t *__restrict__ out_ids, double *__restrict__ out_dist,
               uint32_t *__restrict__ out_count) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    uint64_t *bkey = (uint64_t *)smem_raw;   // [256]
    uint64_t *tkey = bkey + 256;              // [k]
    uint32_t *bid = (uint32_t *)(tkey + k);   // [256]
    uint32_t *tid_ = bid + 256;               // [k]
    uint32_t *ctl = tid_ + k;                 // [1]
    const int tid = threadIdx.x;
    const uint32_t b = blockIdx.x;
    const size_t total = (size_t)n_parts * k, at = (size_t)b * total;
    int tcnt = 0, fill = 0;
    if (tid == 0) ctl[0] = 0;
    __syncthreads();
    for (size_t e0 = 0; e0 < total; e0 += 256) {
        // entries that can still enter the list are gathered until 256 could overflow the batch
        const size_t e = e0 + tid;
        uint64_t key = ~0ull;
        uint32_t id = CZ_NONE;
        if (e < total) {
            key = part_key[at + e];
            id = part_id[at + e];
        }
        const bool want = id != CZ_NONE && (tcnt < (int)k || czh::key_lt(key, id, tkey[k - 1], tid_[k - 1]));
        const int add = __syncthreads_count(want);
        if (fill + add > 256) {
            tcnt = topk_merge_batch(fill, bkey, bid, tkey, tid_, tcnt, (int)k);
            if (tid == 0) ctl[0] = 0;
            fill = 0;
            __syncthreads();
        }
        if (want) {
            const uint32_t p = atomicAdd(&ctl[0], 1u);  // (the order within a batch does not matter: entries are ranked)
            bkey[p] = key;
            bid[p] = id;
        }
        fill += add;
    }
    tcnt = topk_merge_batch(fill, bkey, bid, tkey, tid_, tcnt, (int)k);
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
uint32_t lanes_per_row(uint32_t chunks) {
    uint32_t l = 4;
    while (l < chunks && l < 64) l <<= 1;
    return l;
}
#define CZ_Q4_LANES(LPR, CALL)      \
    switch (LPR) {                  \
        case 4: CALL(4); break;     \
        case 8: CALL(8); break;     \
        case 16: CALL(16); break;   \
        case 32: CALL(32); break;   \
        default: CALL(64); break;   \
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

struct KnnPlan {
    uint32_t chunks, tiles_per_chunk;
    uint64_t *part_key;
    uint32_t *part_id;
    size_t bytes;
};
KnnPlan knn_plan(const Rows &t, uint32_t B, uint32_t k, void *ws) {
    KnnPlan p;
    const uint32_t n_tiles = (t.n + kTile - 1) / kTile;
    // 256 rows are a batch of the list; enough workgroups to fill the chip, few enough lists to join
    uint32_t chunks = std::min((n_tiles + 3) / 4, std::max(1u, 2048 / B));
    chunks = std::max(1u, std::min(chunks, std::max(16u, 65536 / k)));
    p.tiles_per_chunk = std::max(1u, (n_tiles + chunks - 1) / chunks);
    p.tiles_per_chunk = (p.tiles_per_chunk + 3) & ~3u;
    p.chunks = std::max(1u, (n_tiles + p.tiles_per_chunk - 1) / p.tiles_per_chunk);
    cz::Carve c(ws);
    p.part_key = c.take<uint64_t>((size_t)B * p.chunks * k);
    p.part_id = c.take<uint32_t>((size_t)B * p.chunks * k);
    p.bytes = c.used();
    return p;
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
#define CZ_Q4_CALL(L)                                                                                                              \
    if (elem == CZ_ELEM_F32)                                                                                                       \
        hipLaunchKernelGGL((q4_quantize_kernel<float, L>), dim3((n + 256 / L - 1) / (256 / L)), dim3(256), 0, stream,              \
                           (const float *)x, ld, wide, t, codes, scales, sqnorms);                                                 \
    else                                                                                                                           \
        hipLaunchKernelGGL((q4_quantize_kernel<uint16_t, L>), dim3((n + 256 / L - 1) / (256 / L)), dim3(256), 0, stream,           \
                           (const uint16_t *)x, ld, wide, t, codes, scales, sqnorms)
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
    return k ? std::max<size_t>(256, knn_plan(t, std::min(B, kMaxBatch), k, nullptr).bytes) : 256;
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
    const uint32_t lpr = lanes_per_row(t.chunks);
#define CZ_Q4_CALL(L)                                                                                                            \
    hipLaunchKernelGGL((q4_dots_kernel<L>), dim3((n + 256 / L - 1) / (256 / L)), dim3(256), 0, stream, t, queries, B, out)
    CZ_Q4_LANES(lpr, CZ_Q4_CALL);
#undef CZ_Q4_CALL
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
    const size_t smem = 256 * 12 + (size_t)k * 12 + 32 + (size_t)dim * 4;
    const uint32_t lpr = lanes_per_row(t.chunks);
    for (uint32_t b0 = 0; b0 < B; b0 += kMaxBatch) {
        const uint32_t nb = std::min(kMaxBatch, B - b0);
        const float *q = queries + (size_t)b0 * dim;
        KnnPlan p{};
        if (n) {
            p = knn_plan(t, nb, k, base);
#define CZ_Q4_CALL(L)                                                                                                              \
    hipLaunchKernelGGL((q4_scan_kernel<L>), dim3(p.chunks, nb), dim3(256), smem, stream, metric, t, q, k, p.tiles_per_chunk,       \
                       p.part_key, p.part_id)
            CZ_Q4_LANES(lpr, CZ_Q4_CALL);
#undef CZ_Q4_CALL
        }
        hipLaunchKernelGGL(q4_join_kernel, dim3(nb), dim3(256), 256 * 12 + (size_t)k * 12 + 16, stream, p.part_key, p.part_id, p.chunks, k,
                           has_radius, radius, out_ids + (size_t)b0 * k, out_dist + (size_t)b0 * k, out_count + b0);
    }
    rc = launched("cz_q4_knn");
    if (rc) return rc;
    if (!dev) return stage.finish();
    if (own.p) CZ_HIP(hipStreamSynchronize(stream));
    return CZ_OK;
}
