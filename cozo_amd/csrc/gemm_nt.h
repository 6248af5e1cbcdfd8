// gemm_nt.h -- the matrix-core loop that the dense operators share:  C[m][n] = sum_k A[m][k] * B[n][k],  operands with k contiguous
// or (16-bit types) with rows contiguous.  A workgroup owns a BM x BN tile; what happens to the accumulators is the caller's epilogue.
//
// * k goes in steps of 128 bytes per row (64 bf16 / 32 f32): a step of A and B goes straight from memory into LDS (16 bytes a lane, no
//   registers in between), two steps are kept, the next one is on its way while the matrix cores work on this one.
// * LDS rows are 128 bytes = 8 pieces of 16; piece p of row r lies at place p ^ (r / 2 & 7): two rows fill the 64 banks, so 16 neighbouring
//   rows read at one k touch each bank once (p ^ (r & 7), which 32 banks would ask for, counted as many conflicts as reads).  The copy into LDS writes lanes in order, so it is the lane's GLOBAL address that is permuted.
// * operand layout of the 32 x 32 matrix instructions: lane l holds row l % 32 and the k that belong to half l / 32; as both
//   operands are read alike, which k those are does not matter: a half is a 16-byte piece (8 bf16 = one 32x32x16 instruction, 4 f32 =
//   four 32x32x2 ones).
// * a turned operand lies in LDS as it does in memory, k by k: a k's rows in pieces of 16 bytes (8 rows), piece p at place p ^ 4 (k & 3)
//   (64 rows: p ^ 4 (k / 2 & 1)).  The
//   transposing read gives 16 lanes of 8 bytes (4 rows) at 4 k's back as 16 rows at 4 k's; 32 lanes read 64 bytes at each of 4 k's, each
//   in a quarter of the banks of its own.
// * accumulators: register r of lane l is C[8 (r / 4) + 4 (l / 32) + r % 4][l % 32] of its 32 x 32 tile.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace gemm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
    static constexpr int kPerPiece = 1;  // matrix instructions of a 16-byte piece
    typedef __bf16 T;
    static constexpr uint32_t kStep = 64;  // elements of a 128-byte step
};
struct F16 {
    static constexpr int kPerPiece = 1;
    typedef _Float16 T;
    static constexpr uint32_t kStep = 64;
};
struct F32 {
    static constexpr int kPerPiece = 4;
    typedef float T;
    static constexpr uint32_t kStep = 32;
};

__device__ __forceinline__ void mma(Bf16, const u32x4 &a, const u32x4 &b, f32x16 &c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(F16, const u32x4 &a, const u32x4 &b, f32x16 &c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(F32, const u32x4 &a, const u32x4 &b, f32x16 &c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
}

// Workgroups go round the 8 XCDs.  The place of this one in an order that gives each XCD a run of neighbours, which read the same rows through
// its L2.
__device__ __forceinline__ uint32_t place_in_order() {
    const uint32_t x = blockIdx.x % 8, per = gridDim.x / 8, rest = gridDim.x % 8;
    return x * per + min(x, rest) + blockIdx.x / 8;
}

// rows of one operand as a workgroup sees them, 16-byte aligned; rows past the last one are read as the last one (the epilogue drops them)
struct Operand {
    const char *base;
    uint64_t ld;            // bytes from a row to the next
    uint32_t rows;
    uint64_t step = 128;    // bytes from a step of k to the next: 128 in ordinary rows, more where k is cut into panels
};
// ordinary rows of `bytes` bytes (a multiple of 16), read where they are although a step ends behind them: it gets zeros there
struct Tailed {
    Operand rows_of;
    uint32_t rows, bytes;
};
// rows of `bytes` bytes at any place: no 16 bytes of them need be aligned to more than an element T
template <typename T>
struct Ragged {
    Operand rows_of;
    uint32_t rows, bytes;
};
// an operand of a 16-bit type that lies turned: for each k the rows one behind the other
struct Turned {
    const char *base;
    uint64_t ld;            // bytes from a k to the next
    uint64_t panel;         // bytes from 64 rows to the next 64: 128 where a k's rows are one run
    uint32_t rows, ks;      // rows: a multiple of 8, 16-byte aligned; a k past the last one is read as the last one (times zeros of the other side)
};
// k in panels: a step's 128 bytes of every row lie one behind the other, so that a workgroup's step is one run of memory; in rows of 128 KB each
// row of a step begins in the same few memory channels (grad_queries of a 65536-row piece: 179 us, with padded rows 168, in panels 164)
inline Operand panels(const void *base, uint32_t rows) { return Operand{(const char *)base, 128, rows, (uint64_t)rows * 128}; }

typedef short s16x4 __attribute__((ext_vector_type(4)));

static __device__ const u32x4 kZeros = {0, 0, 0, 0};

// a workgroup's copies of ROWS rows of an operand into LDS, a step at a time
template <class O, int ROWS, int THREADS>
struct Copies;
template <int ROWS, int THREADS>
struct Copies<Operand, ROWS, THREADS> {
    static constexpr int N = ROWS * 8 / THREADS;  // 16-byte pieces of a thread
    static constexpr bool kHeld = false;           // copies go straight into LDS
    static constexpr int kReads = 1;               // LDS reads of a fragment
    static_assert(N * THREADS == ROWS * 8, "threads cover the copies");
    const char *src[N];
    uint64_t stride;
    static __device__ __forceinline__ uint32_t piece(int i) {  // (of the step's 128 bytes)
        const uint32_t c = i * THREADS + threadIdx.x;
        return ((c & 7) ^ ((c >> 4) & 7)) * 16;
    }
    __device__ __forceinline__ Copies(const Operand &o, uint32_t row0) : stride(o.step) {
#pragma unroll
        for (int i = 0; i < N; i++) src[i] = o.base + (uint64_t)min(row0 + (i * THREADS + threadIdx.x) / 8, o.rows - 1) * o.ld;
    }
    __device__ __forceinline__ const char *from(int i, uint32_t step) const { return src[i] + (step * stride + piece(i)); }
    // rows row0 + 32 i + lane % 32 at the 16 k's `kk` of a step
    static __device__ __forceinline__ u32x4 fragment(const char *lds, int row0, int i, int kk) {
        const int lane = threadIdx.x & 63, l32 = lane & 31;
        return *(const u32x4 *)(lds + (row0 + l32) * 128 + (((2 * kk + (lane >> 5)) ^ ((l32 >> 1) & 7)) * 16) + i * 32 * 128);
    }
};
// (a kernel of its own for rows that end inside a step: the comparison in every copy took 10 % of the products that do not need it)
template <int ROWS, int THREADS>
struct Copies<Tailed, ROWS, THREADS> : Copies<Operand, ROWS, THREADS> {
    uint32_t bytes;
    __device__ __forceinline__ Copies(const Tailed &o, uint32_t row0) : Copies<Operand, ROWS, THREADS>(o.rows_of, row0), bytes(o.bytes) {}
    __device__ __forceinline__ const char *from(int i, uint32_t step) const {
        const uint32_t at = step * 128 + this->piece(i);
        return at < bytes ? this->src[i] + at : reinterpret_cast<const char *>(&kZeros);
    }
};
// Through registers: the copy into LDS asks for aligned dwords.  A step's loads are on their way while the step before it is worked on.  What
// ends in a row's last step is read an element at a time, no further than the row.
// (7 queries, 349365 rows of 1011 in f32: 322 us; packed into aligned rows first, 1315)
template <typename T, int ROWS, int THREADS>
struct Copies<Ragged<T>, ROWS, THREADS> : Copies<Operand, ROWS, THREADS> {
    typedef Copies<Operand, ROWS, THREADS> Base;
    static constexpr bool kHeld = true;
    uint32_t bytes;
    u32x4 held[Base::N];
    __device__ __forceinline__ Copies(const Ragged<T> &o, uint32_t row0) : Base(o.rows_of, row0), bytes(o.bytes) {}
    __device__ __forceinline__ void fetch(uint32_t step) {
        if ((step + 1) * 128 <= bytes) {
#pragma unroll
            for (int i = 0; i < Base::N; i++) __builtin_memcpy(&held[i], this->src[i] + (step * 128 + this->piece(i)), 16);
        } else {
            constexpr uint32_t P = 16 / sizeof(T);
            typedef T Piece __attribute__((ext_vector_type(P)));
#pragma unroll
            for (int i = 0; i < Base::N; i++) {
                const uint32_t at = step * 128 + this->piece(i);
                Piece x;
#pragma unroll
                for (uint32_t j = 0; j < P; j++) {
                    x[j] = (T)0.f;
                    if (at + j * sizeof(T) < bytes) x[j] = *(const T *)(this->src[i] + at + j * sizeof(T));
                }
                held[i] = __builtin_bit_cast(u32x4, x);
            }
        }
    }
    __device__ __forceinline__ void put(char *lds) const {
#pragma unroll
        for (int i = 0; i < Base::N; i++) *(u32x4 *)(lds + (i * THREADS + threadIdx.x) * 16) = held[i];
    }
};
template <int ROWS, int THREADS>
struct Copies<Turned, ROWS, THREADS> {
    static constexpr bool kHeld = false;
    static constexpr int N = ROWS * 8 / THREADS, P = ROWS / 8;  // pieces of a thread, of a k
    static constexpr int kReads = 2;
    static_assert(N * THREADS == ROWS * 8, "threads cover the copies");
    static_assert(P >= 8, "a k's rows fill half of the banks at least");
    // what a k's pieces are placed by (64 rows: two k's fill the banks)
    static __device__ __forceinline__ uint32_t turn(uint32_t k) { return P >= 16 ? 4 * (k & 3) : 4 * ((k >> 1) & 1); }
    const char *src[N];
    uint64_t ld;
    uint32_t ks;
    __device__ __forceinline__ Copies(const Turned &o, uint32_t row0) : ld(o.ld), ks(o.ks) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t c = i * THREADS + threadIdx.x, k = c / P, piece = (c % P) ^ turn(k);
            const uint32_t row = min(row0 + piece * 8, o.rows - 8);
            src[i] = o.base + (row >> 6) * o.panel + (row & 63) * 2;
        }
    }
    __device__ __forceinline__ const char *from(int i, uint32_t step) const {
        const uint32_t k = step * 64 + (i * THREADS + threadIdx.x) / P;
        return src[i] + min(k, ks - 1) * ld;
    }
    static __device__ __forceinline__ u32x4 fragment(const char *lds, int row0, int i, int kk) {
        const int lane = threadIdx.x & 63, l16 = lane & 15;
        const int k = 16 * kk + 8 * (lane >> 5) + (l16 >> 2), col = row0 + i * 32 + 16 * ((lane >> 4) & 1) + 4 * (l16 & 3);
        const int at = ((col >> 3) ^ turn(l16 >> 2)) * 16 + (col & 7) * 2;
        typedef __attribute__((address_space(3))) s16x4 *Lds;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(lds + k * P * 16 + at)),
                    b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(lds + (k + 4) * P * 16 + at));
        struct {
            s16x4 a, b;
        } both = {a, b};
        return __builtin_bit_cast(u32x4, both);
    }
};

// BM x BN by WM x WN waves.  Measured with 1024 rows of B, 1M rows of A, k = 768, bf16, products alone: 128 x 128 by 2 x 2 900 TFLOP/s (32 bytes of
// copies a clock and CU), 256 x 256 by 2 x 4 1185 (a library's 8192^3 product: 1537).  With its epilogue the forward product of the softmax runs at 1060,
// its matrix cores busy 49 % of the time by their counter, the gradient's at 690 to 770 (29 to 33 %); no LDS bank conflicts in any.  Zeros for data run at
// 1310: the clock under this load is part of the bound.  More and shorter steps kept in LDS, tiles run into each other and a wave priority for the
// matrix instructions were within 5 % of it either way.
template <class E, int BM_, int BN_, int WM_, int WN_>
struct Tile {
    typedef E Elem;
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
    static constexpr int kThreads = 64 * WM * WN;
    static constexpr int MT = BM / WM / 32, NT = BN / WN / 32;
    static constexpr int kBytes = (BM + BN) * 128;  // LDS of one step
    static constexpr int kLds = 2 * kBytes;
    static_assert(MT * WM * 32 == BM && NT * WN * 32 == BN, "waves cover the tile");

    // f32: a step's four quarters go to sums of their own as far as registers allow, joined at the end: a shorter chain of additions rounds less
    // (dW of 1 query x 3001 rows x 640: 1.2e-6 off with one sum, 0.6e-6 with four; the time is the same)
    static constexpr int kChains = E::kPerPiece == 1 || MT * NT > 4 ? 1 : MT * NT == 1 ? 4 : 2;

    f32x16 acc[MT][NT];
    f32x16 more[kChains > 1 ? kChains - 1 : 1][MT][NT];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    acc[i][j][r] = 0.f;
#pragma unroll
                    for (int c = 1; c < kChains; c++) more[c - 1][i][j][r] = 0.f;
                }
    }
    typedef Copies<Operand, BM, kThreads> CopiesA;
    typedef Copies<Operand, BN, kThreads> CopiesB;
    template <class C>
    static __device__ __forceinline__ void copy(const C &c, uint32_t step, char *lds) {
        const uint32_t wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < C::N; i++)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)c.from(i, step),
                                             (__attribute__((address_space(3))) void *)(lds + (i * kThreads + wave * 64) * 16), 16, 0, 0);
    }
    // the copies this wave has in flight are in LDS, and every wave is here
    static __device__ __forceinline__ void arrived() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    static __device__ __forceinline__ int wave_row() { return (int)(threadIdx.x >> 6) / WN * (BM / WM); }
    static __device__ __forceinline__ int wave_col() { return (int)(threadIdx.x >> 6) % WN * (BN / WN); }

    template <class CA, class CB>
    static __device__ __forceinline__ void fragments(const char *lds, int kk, u32x4 (&a)[MT], u32x4 (&b)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; j++) b[j] = CB::fragment(lds + BM * 128, wave_col(), j, kk);
#pragma unroll
        for (int i = 0; i < MT; i++) a[i] = CA::fragment(lds, wave_row(), i, kk);
    }
    template <class CA = CopiesA, class CB = CopiesB>
    __device__ __forceinline__ void step(const char *lds) {
        u32x4 a[2][MT], b[2][NT];
        fragments<CA, CB>(lds, 0, a[0], b[0]);
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            if (kk < 3) fragments<CA, CB>(lds, kk + 1, a[(kk + 1) & 1], b[(kk + 1) & 1]);
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) mma(E{}, a[kk & 1][i], b[kk & 1][j], kk % kChains ? more[kk % kChains - 1][i][j] : acc[i][j]);
        }
        // the next fragments are read between this fragment's matrix instructions
        constexpr int R = MT * CA::kReads + NT * CB::kReads, X = MT * NT, PER = (R + X - 1) / X;
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
#pragma unroll
        for (int kk = 0; kk < 4; kk++)
#pragma unroll
            for (int x = 0; x < X; x++) {
                if (kk < 3 && x * PER < R) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, E::kPerPiece, 0);
            }
    }
    // one tile: A rows from m0, B rows from n0, `steps` >= 1 steps from step s0 on
    template <class OA, class OB>
    __device__ __forceinline__ void run(const OA &A, uint32_t m0, const OB &B, uint32_t n0, uint32_t s0, uint32_t steps, char *lds) {
        typedef Copies<OA, BM, kThreads> CA;
        typedef Copies<OB, BN, kThreads> CB;
        CA ca(A, m0);
        const CB cb(B, n0);
        zero();
        copy(cb, s0, lds + BM * 128);
        if constexpr (CA::kHeld) {
            ca.fetch(s0);
            ca.put(lds);
        } else copy(ca, s0, lds);
        for (uint32_t s = 0; s < steps; s++) {
            char *cur = lds + (s & 1) * kBytes, *nxt = lds + (~s & 1) * kBytes;
            arrived();
            if (s + 1 < steps) {
                if constexpr (CA::kHeld) ca.fetch(s0 + s + 1);
                else copy(ca, s0 + s + 1, nxt);
                copy(cb, s0 + s + 1, nxt + BM * 128);
            }
            step<CA, CB>(cur);
            if constexpr (CA::kHeld)
                if (s + 1 < steps) ca.put(nxt);
        }
#pragma unroll
        for (int c = 1; c < kChains; c++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] += more[c - 1][i][j];
    }
    // f(row, col, value) over this thread's accumulators, rows and columns within the tile
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    f(wave_row() + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), wave_col() + j * 32 + (lane & 31), acc[i][j][r]);
    }
};

}  // namespace gemm
