// Pieces of the gated delta rule's kernels: operands as terms of bf16, tiles in shared memory, fragments of mma.sync.
//
// A value is taken as one to three bf16 terms (8 bits each: x = hi + mid + lo), a product of two values as the products of their
// terms i and j with i + j < N, N the terms that the result deserves: 2^-9, 2^-17 or 2^-24 of each product is dropped. bf16 values
// are one term as they are, fp16 values two. (mma.sync of tf32 takes twice the time of bf16 for the same product: two bf16 terms
// cost as much as one of tf32 and keep 16 bits instead of 11.)
//
// mma.sync m16n8k16: a thread (g = lane / 4, t4 = lane % 4) of the warp has of a 16 x 8 result the values (g, 2 t4), (g, 2 t4 + 1),
// (g + 8, 2 t4), (g + 8, 2 t4 + 1); two such results side by side are, packed in pairs, the 16 x 16 left operand of the next product.
#pragma once
#include "fg_heads.cuh"

namespace {
using namespace fgm;
using bf16 = __nv_bfloat16;

constexpr int kTicks = 64;               // of a slot: where states are kept for the gradients
constexpr int kChunk = 32;               // of a chunk of the chain, two to a slot
constexpr int kSquare = kTicks + 8;      // a row of a 64 x 64 tile in shared memory: 8 rows of 16 bytes lie in 32 banks
constexpr int kSmall = kChunk + 8;       // and of a 32 x 32 one

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (volatile: they stay between the barriers around them; loads from global memory may pass them)
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ void stsm_t(uint32_t at, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// the product without a sum before it
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// a pair of values as N packed terms
template <int N>
__device__ __forceinline__ void terms(float x, float y, uint32_t (&t)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        t[i] = pack(x, y);
        if (i + 1 < N) {
            x -= low(t[i]);
            y -= high(t[i]);
        }
    }
}
// two 16 x 8 results side by side as a left operand of N terms
template <int N>
__device__ __forceinline__ void left(const float (&x)[4], const float (&y)[4], uint32_t (&a)[N][4]) {
    const float* v[4] = {&x[0], &x[2], &y[0], &y[2]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t t[N];
        terms<N>(v[i][0], v[i][1], t);
#pragma unroll
        for (int n = 0; n < N; ++n) a[n][i] = t[n];
    }
}

// Where a lane's 16 bytes of four 8 x 8 blocks lie in a tile with rows of `stride` values (a byte offset):
// right operand from rows n of values k: blocks (n 0-7, k 0-7), (n 0-7, k 8-15), (n 8-15, k 0-7), (n 8-15, k 8-15)
__device__ __forceinline__ uint32_t at_rows_n(int lane, int stride) { return 2 * (((lane & 7) + ((lane >> 4) << 3)) * stride + ((lane >> 3) & 1) * 8); }
// left operand from rows m of values k, or (transposed) right operand from rows k of values n:
// blocks (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
__device__ __forceinline__ uint32_t at_rows_m(int lane, int stride) { return 2 * ((lane & 15) * stride + (lane >> 4) * 8); }
// transposed: left operand from rows k of values m: the same blocks as at_rows_n
__device__ __forceinline__ uint32_t at_rows_k(int lane, int stride) { return at_rows_n(lane, stride); }

struct Operand {
    char* p;
    long long batch, tick, head;
    int share;               // heads to one head of this operand
    int fast;                // whole 16 bytes of 8 values (32 of fp32) at 16-byte boundaries
};
struct Gate {
    float* p;
    long long batch, tick, head;
};
struct Span {
    long long start, n;      // ticks of the recording
};

__device__ __forceinline__ void async16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows 0 .. ROWS - 1 of an operand (`rows` of them there, the rest zeros), columns 0 .. COLS - 1 of `cols`, as N planes of terms
// with rows of STRIDE values. bf16 at 16-byte boundaries goes by asynchronous copies.
template <class T, int N, int COLS, int STRIDE, int THREADS, int ROWS = kTicks>
__device__ __forceinline__ void load_tile(bf16* to, const T* p, long long row, int rows, int cols, bool fast, int tid) {
    constexpr int kUnits = COLS / 8, kPlane = ROWS * STRIDE, kStep = THREADS / kUnits;
    static_assert(THREADS % kUnits == 0 && ROWS % kStep == 0, "a thread keeps its columns");
    const int r0 = tid / kUnits, c = tid % kUnits * 8;
    const bool has = c < cols;
    const T* q = p + (has ? r0 * row + c : 0);
    bf16* at = to + r0 * STRIDE + c;
#pragma unroll 4
    for (int r = r0; r < ROWS; r += kStep, q += kStep * row, at += kStep * STRIDE) {
        const bool in = has && r < rows;
        if constexpr (N == 1 && std::is_same<T, bf16>::value) {
            if (fast) {
                async16(smem_at(at), in ? q : p, in);
                continue;
            }
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (in) {
            if (fast) {
                constexpr int kLoads = 8 * (int)sizeof(T) / 16;
                uint4 u[kLoads];
#pragma unroll
                for (int j = 0; j < kLoads; ++j) u[j] = reinterpret_cast<const uint4*>(q)[j];
                const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = to_f(e[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < cols) x[j] = to_f(q[j]);
            }
        }
        uint32_t t[4][N];
#pragma unroll
        for (int j = 0; j < 4; ++j) terms<N>(x[2 * j], x[2 * j + 1], t[j]);
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<uint4*>(at + n * kPlane) = make_uint4(t[0][n], t[1][n], t[2][n], t[3][n]);
    }
}
// N planes of a 32 x 32 tile from the workspace (rows of 32) to rows of kSmall
template <int N, int THREADS>
__device__ __forceinline__ void load_small(bf16* to, const bf16* p, int tid) {
    for (int i = tid; i < N * kChunk * 4; i += THREADS) async16(smem_at(to + (i >> 2) * kSmall + (i & 3) * 8), p + i * 8, true);
}

// 8 sums over the 8 lanes g with the same t4, of v[2 j + i] = a value of column 8 j + 2 t4 + i: lane g keeps column 8 (g / 2) + 2 t4 + g % 2
__device__ __forceinline__ float column_sums(float (&v)[8], int lane) {
#pragma unroll
    for (int half = 4; half >= 1; half >>= 1) {
        const int bit = half * 4;                            // lanes 16, 8, 4 apart
        const bool upper = lane & bit;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
        }
    }
    return v[0];
}

// Terms by type: of inputs; of all that is carried from chunk to chunk and what corrects it (states, X, their gradients); of S and of P
// and U where they make o; for the gradients of q and k of U, dP and D, of S, of R, and of dN.
// Three terms keep states, their gradients and the gates' as good as fp32 products and sums would (64 recordings of 1,024 ticks, 8 heads of
// 128 in bf16: 3e-7 to 7e-7 off; with two terms 4e-6 to 1e-5, in 360 instead of 497 us for the chain forward). o and the gradients of
// q and k are rounded to 16 bits in the end, 1.65e-3 of their norm. With P, U and S of one term they were up to 3.1e-3 off (o of short
// recordings, nearly all P U), with R and dN of one gk 2.3e-3; with these terms o, gq and gk are as good as their rounding (o 522 instead of
// 501 us; gradients with R and dN of one term 893 instead of 1,032, the way back to them 965 instead of 1,015).
template <class T> struct Terms;
template <> struct Terms<bf16> { static constexpr int in = 1, kept = 3, out_s = 2, out_p = 2, grad = 2, grad_s = 2, grad_r = 2, grad_n = 2; };
template <> struct Terms<__half> { static constexpr int in = 2, kept = 3, out_s = 2, out_p = 2, grad = 2, grad_s = 2, grad_r = 2, grad_n = 2; };
template <> struct Terms<float> { static constexpr int in = 3, kept = 3, out_s = 3, out_p = 3, grad = 3, grad_s = 3, grad_r = 3, grad_n = 3; };

// sum[2 J] += a b for J pairs of 8 x 16 right operands from planes of NB terms at(j, pair), products with term numbers below KEEP; term
// by term over all pairs, so that no product waits for the one just before. `first`: sum = a b. The tensor cores cut sums off, they do not
// round them: where both operands have terms (so many products) the small ones are added up first, by themselves, and their sum with the
// large one to `sum` in fp32 (1.0e-6 to 2.1e-6 off without that, 4e-7 to 7e-7 with it, 32 recordings of 509 ticks, 4 heads of 64 in fp32).
template <int NA, int NB, int KEEP, int J, bool TRANS, class At>
__device__ __forceinline__ void products(float (*sum)[4], const uint32_t (&a)[NA][4], At&& at, bool first = false) {
    if constexpr (KEEP >= 3 && NB >= 2) {
        uint32_t r[NB][J][4];
        float x[2 * J][4];
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int p = 0; p < J; ++p) {
                if (TRANS) ldsm_t(r[j][p], at(j, p));
                else ldsm(r[j][p], at(j, p));
            }
        constexpr int most = NA + NB - 2 < KEEP - 1 ? NA + NB - 2 : KEEP - 1;
#pragma unroll
        for (int s = most; s >= 0; --s)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int k = s - j;
                if (k < 0 || k >= NA) continue;
                const bool opens = s == most && (j == 0 || k == NA - 1);   // the first of all
#pragma unroll
                for (int p = 0; p < J; ++p) {
                    if (opens) {
                        mma_first(x[2 * p], a[k], r[j][p][0], r[j][p][1]);
                        mma_first(x[2 * p + 1], a[k], r[j][p][2], r[j][p][3]);
                    } else {
                        mma(x[2 * p], a[k], r[j][p][0], r[j][p][1]);
                        mma(x[2 * p + 1], a[k], r[j][p][2], r[j][p][3]);
                    }
                }
            }
#pragma unroll
        for (int p = 0; p < 2 * J; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[p][e] = first ? x[p][e] : sum[p][e] + x[p][e];
    } else {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            uint32_t r[J][4];
#pragma unroll
            for (int p = 0; p < J; ++p) {
                if (TRANS) ldsm_t(r[p], at(j, p));
                else ldsm(r[p], at(j, p));
            }
#pragma unroll
            for (int k = 0; k < NA && k + j < KEEP; ++k)
#pragma unroll
                for (int p = 0; p < J; ++p) {
                    if (first && j + k == 0) {
                        mma_first(sum[2 * p], a[k], r[p][0], r[p][1]);
                        mma_first(sum[2 * p + 1], a[k], r[p][2], r[p][3]);
                    } else {
                        mma(sum[2 * p], a[k], r[p][0], r[p][1]);
                        mma(sum[2 * p + 1], a[k], r[p][2], r[p][3]);
                    }
                }
        }
    }
}

}  // namespace
