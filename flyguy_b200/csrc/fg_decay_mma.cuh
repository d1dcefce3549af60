// The decay scan of fp32 and fp16 operands (and of bf16 ones whose sizes or strides the TMA tiles do not fit), dim and
// value_dim up to 128: chunks of 64 ticks as products of tf32 terms (mma.sync m16n8k8, fp32 sums).
//
//   W = (a b^T) . gamma^{t-s},  out = scale_out (gamma^{t+1} a S + W c),  S <- gamma^n S + b'^T c,  b' = scale_in gamma^{n-1-s} b
//
// An fp32 value is taken as hi + lo, both tf32 (11 bits each), and a product as hi hi + hi lo + lo hi: 2^-21 of each
// product is dropped, about the rounding of the fp32 sums. 16-bit inputs are tf32 values as they are (lo = 0), so only S,
// W and b' have two terms there. The tensor cores cut their sums off rather than round them, always towards zero: products of
// hi parts are summed 32 deep, then added on in fp32, those with lo parts by themselves (1,500 ticks in one accumulator came
// to 5e-6 of S). S stays in the fp32 accumulators of the warps; a copy in shared memory is the next
// chunk's operand. Tensor instructions that reach further (tcgen05 kind::tf32) want operands of 4 bytes a value split
// beforehand, two planes each: at dim 128 one chunk's would not fit beside S in 227 KB.
//
// A NaN or an infinity reaches all ticks of its chunk, and an infinity becomes a NaN in its terms (hi infinite, lo not a number).
//
// 32 recordings of 509 ticks, 4 heads of 64 in fp32: 131 us a scan (52 MB in; 6.4 GFLOP as 3 products of terms), 379 us forward and
// back, the three scans back overlapping. Bound by waits: 8 warps of a block share the four products of a chunk, with a
// barrier between each, and a block or two share an SM; the tensor pipe is 14% busy, issue slots 21%, DRAM 5%.
#pragma once
#include "fg_memory.cuh"

namespace {
using namespace fgm;

constexpr int kMmTicks = 64, kMmThreads = 256;

__device__ __forceinline__ void mma_tf32_sync(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t tf32_of(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
// n values as terms: hi, and lo (what is left; the tensor cores drop its last bits)
template <int N>
__device__ __forceinline__ void split_tf32(const float (&x)[N], uint32_t (&hi)[N], uint32_t (&lo)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        hi[i] = tf32_of(x[i]);
        lo[i] = __float_as_uint(x[i] - __uint_as_float(hi[i]));
    }
}

__device__ __forceinline__ void zero(float (&d)[4][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
}
__device__ __forceinline__ void add(float (&d)[4][4], const float (&x)[4][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[j][i] += x[j][i];
}
// sum[16 x 32] += a b over k0 .. k1 - 1 (multiples of 8); a4(k) and b2(k, j) give a fragment's values
// of a 16 x 8 and the j-th 8 x 8 block; which of the two are tf32 values as they are; alive(j): blocks that count
template <bool EXACT_A, bool EXACT_B, class A, class B, class L>
__device__ __forceinline__ void products(float (&sum)[4][4], int k0, int k1, A&& a4, B&& b2, L&& alive) {
    float low[4][4];
    zero(low);
#pragma unroll 1
    for (int kk = k0; kk < k1; kk += 32) {
        float high[4][4];
        zero(high);
#pragma unroll 1
        for (int k = kk; k < min(kk + 32, k1); k += 8) {
            float x[4];
            a4(k, x);
            uint32_t hi[4], lo[4];
            if (EXACT_A) {
#pragma unroll
                for (int i = 0; i < 4; ++i) hi[i] = __float_as_uint(x[i]);
            } else {
                split_tf32(x, hi, lo);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!alive(j)) continue;
                float y[2];
                b2(k, j, y);
                uint32_t bh[2] = {__float_as_uint(y[0]), __float_as_uint(y[1])}, bl[2];
                if (!EXACT_B) {
                    split_tf32(y, bh, bl);
                    mma_tf32_sync(low[j], hi, bl);
                }
                if (!EXACT_A) mma_tf32_sync(low[j], lo, bh);
                mma_tf32_sync(high[j], hi, bh);
            }
        }
        add(sum, high);
    }
    if (!EXACT_A || !EXACT_B) add(sum, low);
}

template <int DP, int EP>
struct MmLayout {                                            // strides that spread a fragment's reads over the banks
    static constexpr int ab = DP + 4, c = EP + 8, w = kMmTicks + 4;
    static constexpr int a0 = 0, b0 = a0 + kMmTicks * ab, c0 = b0 + kMmTicks * ab, s0 = c0 + kMmTicks * c, w0 = s0 + DP * c,
                         pw0 = w0 + kMmTicks * w, floats = pw0 + kMmTicks + 4;
};

// EXACT: operands of 16 bits; PARTS: the states of the parts alone
template <class T, int DP, int EP, bool BACK, bool PARTS>
__global__ void __launch_bounds__(kMmThreads, DP + EP < 256 ? 2 : 1) k_decay_mma(const __grid_constant__ Scan s, int quads) {
    extern __shared__ __align__(16) float mm[];
    using L = MmLayout<DP, EP>;
    constexpr bool EXACT = sizeof(T) == 2;
    float *sa = mm + L::a0, *sb = mm + L::b0, *sc = mm + L::c0, *ss = mm + L::s0, *sw = mm + L::w0, *pw = mm + L::pw0;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int D = s.D, E = s.E, h = blockIdx.x % s.heads, part = blockIdx.y;
    const long long b = blockIdx.x / s.heads;
    const Span sp = span_of(s, b);
    const long long per = part_ticks(sp.n, s.parts), t0 = min(sp.n, part * per), t1 = min(sp.n, t0 + per);
    const bool hand_on = !PARTS && s.last && (sp.n ? t1 == sp.n && t1 > t0 : part == 0);
    const bool last_block = s.beside && blockIdx.x == gridDim.x - 1;
    next_may_begin();
    if (t1 == t0 && !hand_on && !PARTS) {
        if (last_block) wait_for_previous();
        return;
    }
    const float ld = s.log_decay[h];
    if (tid <= kMmTicks) pw[tid] = power(ld, (float)tid);

    // a warp's part of S: rows m .. m + 15 of the state, NS blocks of 8 columns
    constexpr int NS = DP == 128 ? EP / 8 : EP / 16;
    const int sm0 = DP == 128 ? warp * 16 : (warp & 3) * 16, sn0 = DP == 128 ? 0 : (warp >> 2) * (EP / 2);
    float S[NS][4];
#pragma unroll
    for (int j = 0; j < NS; ++j) S[j][0] = S[j][1] = S[j][2] = S[j][3] = 0.f;
    const long long state0 = (b * s.heads + h) * D * E;
    // f(row, column, value) over the warp's values
    auto each = [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = sm0 + g + (i >> 1) * 8, e = sn0 + j * 8 + t4 * 2 + (i & 1);
                if (d < D && e < E) f(d, e, S[j][i]);
            }
    };
    if (!PARTS) {
        if (s.first) {
            const float f = power(ld, (float)(BACK ? max(t0 - 1, 0ll) : t0));
            each([&](int d, int e, float& v) { v = f * s.first[state0 + (s.first_t ? (long long)e * D + d : (long long)d * E + e)]; });
        }
        for (int p = 0; p < part; ++p) {
            const float f = power(ld, (float)(t0 - min(sp.n, (p + 1) * per)));
            const float* q = s.partial + ((b * s.heads + h) * s.parts + p) * D * E;
            each([&](int d, int e, float& v) { v = fmaf(f, q[(long long)d * E + e], v); });
        }
    }
    auto put_state = [&]() {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            float* at = ss + (sm0 + g) * L::c + sn0 + j * 8 + t4 * 2;
            *reinterpret_cast<float2*>(at) = make_float2(S[j][0], S[j][1]);
            *reinterpret_cast<float2*>(at + 8 * L::c) = make_float2(S[j][2], S[j][3]);
        }
    };
    if (!PARTS) put_state();

    int lead = BACK && s.first && part == 0 && !PARTS ? 0 : 1;
    for (long long t = t0; t < t1; t += kMmTicks, lead = 1) {
        const int n = (int)min((long long)kMmTicks, t1 - t);
        const long long first = sp.start + (BACK ? sp.n - t - n : t);
        // the tile of an operand, rows in recording order, zeros past its ends
        auto load = [&](const Operand& o, float* to, int stride, int dim, int wide) {
            const T* p = reinterpret_cast<const T*>(o.p) + (s.offsets ? 0 : b * o.batch) + first * o.tick + (h / o.share) * o.head;
            if (quads) {
                for (int i = tid; i < kMmTicks * wide / 4; i += kMmThreads) {
                    const int r = i / (wide / 4), d = (i - r * (wide / 4)) * 4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < n && d < dim) {
                        const T* q = p + (long long)r * o.tick + d;
                        if (sizeof(T) == 4) {
                            v = *reinterpret_cast<const float4*>(q);
                        } else {
                            const uint2 u = *reinterpret_cast<const uint2*>(q);
                            const T* e = reinterpret_cast<const T*>(&u);
                            v = make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
                        }
                    }
                    *reinterpret_cast<float4*>(to + r * stride + d) = v;
                }
            } else {
                for (int i = tid; i < kMmTicks * wide; i += kMmThreads) {
                    const int r = i / wide, d = i - r * wide;
                    to[r * stride + d] = r < n && d < dim ? to_f(p[(long long)r * o.tick + d]) : 0.f;
                }
            }
        };
        __syncthreads();                                      // the chunk before is done with its tiles
        if (!PARTS) load(s.a, sa, L::ab, D, DP);
        load(s.b, sb, L::ab, D, DP);
        load(s.c, sc, L::c, E, EP);
        __syncthreads();
        if (!PARTS) {
            // W: rows m0 .. m0 + 15, columns n0 .. n0 + 31
            const int m0 = (warp & 3) * 16, n0 = (warp >> 2) * 32;
            float acc[4][4];
            zero(acc);
            auto alive = [&](int j) { return BACK ? n0 + j * 8 + 7 >= m0 : n0 + j * 8 <= m0 + 15; };   // meets the diagonal's side
            if (alive(BACK ? 3 : 0))
                products<EXACT, EXACT>(acc, 0, DP,
                    [&](int k, float (&x)[4]) {
                        const float* p = sa + (m0 + g) * L::ab + k + t4;
                        x[0] = p[0]; x[1] = p[8 * L::ab]; x[2] = p[4]; x[3] = p[8 * L::ab + 4];
                    },
                    [&](int k, int j, float (&y)[2]) {
                        const float* p = sb + (n0 + j * 8 + g) * L::ab + k + t4;
                        y[0] = p[0]; y[1] = p[4];
                    }, alive);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = m0 + g + i * 8, c0 = n0 + j * 8 + t4 * 2;
                    const int d0 = BACK ? c0 - r : r - c0, d1 = BACK ? d0 + 1 : d0 - 1;
                    const float f = s.scale_in;
                    const float v0 = d0 >= 0 && (!BACK || c0 < n) ? acc[j][2 * i] * pw[d0 >= 0 ? d0 : 0] * f : 0.f;
                    const float v1 = d1 >= 0 && (!BACK || c0 + 1 < n) ? acc[j][2 * i + 1] * pw[d1 >= 0 ? d1 : 0] * f : 0.f;
                    *reinterpret_cast<float2*>(sw + r * L::w + c0) = make_float2(v0, v1);
                }
            __syncthreads();
            // out: rows m0 .., EP / 2 columns a warp, four blocks of 8 at a time
#pragma unroll 1
            for (int e0 = (warp >> 2) * (EP / 2); e0 < (warp >> 2) * (EP / 2) + EP / 2; e0 += 32) {
                if (e0 >= E) break;
                float o[4][4];
                zero(o);
                auto always = [](int) { return true; };
                products<EXACT, false>(o, 0, DP,
                    [&](int k, float (&x)[4]) {
                        const float* p = sa + (m0 + g) * L::ab + k + t4;
                        x[0] = p[0]; x[1] = p[8 * L::ab]; x[2] = p[4]; x[3] = p[8 * L::ab + 4];
                    },
                    [&](int k, int j, float (&y)[2]) {
                        const float* p = ss + (k + t4) * L::c + e0 + j * 8 + g;
                        y[0] = p[0]; y[1] = p[4 * L::c];
                    }, always);
                const int r0 = m0 + g, r1 = r0 + 8;
                const float f0 = pw[max(BACK ? n - 1 - r0 : r0, 0) + lead], f1 = pw[max(BACK ? n - 1 - r1 : r1, 0) + lead];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
                products<false, EXACT>(o, BACK ? m0 : 0, BACK ? kMmTicks : m0 + 16,
                    [&](int k, float (&x)[4]) {
                        const float* p = sw + (m0 + g) * L::w + k + t4;
                        x[0] = p[0]; x[1] = p[8 * L::w]; x[2] = p[4]; x[3] = p[8 * L::w + 4];
                    },
                    [&](int k, int j, float (&y)[2]) {
                        const float* p = sc + (k + t4) * L::c + e0 + j * 8 + g;
                        y[0] = p[0]; y[1] = p[4 * L::c];
                    }, always);
                const long long at = (s.offsets ? 0 : b * s.out.batch) + first * s.out.tick + h * s.out.head;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = m0 + g + (i >> 1) * 8, e = e0 + j * 8 + t4 * 2 + (i & 1);
                        if (r < n && e < E) {
                            const float v = o[j][i] * s.scale_out;
                            if (s.out_f32) reinterpret_cast<float*>(s.out.p)[at + (long long)r * s.out.tick + e] = v;
                            else reinterpret_cast<T*>(s.out.p)[at + (long long)r * s.out.tick + e] = from_f<T>(v);
                        }
                    }
            }
            __syncthreads();                                  // S's copy has been read
        }
        const float fade = pw[n - 1 + lead];
#pragma unroll
        for (int j0 = 0; j0 < NS; j0 += 4) {
            float d[4][4];
            zero(d);
            products<false, EXACT>(d, 0, (n + 7) / 8 * 8,
                [&](int k, float (&x)[4]) {
                    const int r0 = k + t4, r1 = r0 + 4;
                    const float f0 = r0 < n ? pw[BACK ? r0 : n - 1 - r0] * s.scale_in : 0.f;
                    const float f1 = r1 < n ? pw[BACK ? r1 : n - 1 - r1] * s.scale_in : 0.f;
                    const float* p = sb + r0 * L::ab + sm0 + g;
                    x[0] = p[0] * f0; x[1] = p[8] * f0; x[2] = p[4 * L::ab] * f1; x[3] = p[4 * L::ab + 8] * f1;
                },
                [&](int k, int j, float (&y)[2]) {
                    const float* p = sc + (k + t4) * L::c + sn0 + (j0 + j) * 8 + g;
                    y[0] = p[0]; y[1] = p[4 * L::c];
                }, [](int) { return true; });
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[j0 + j][i] = fmaf(S[j0 + j][i], fade, d[j][i]);
        }
        if (!PARTS) put_state();
    }
    float* to = PARTS ? s.partial + ((b * s.heads + h) * s.parts + part) * D * E : hand_on ? s.last + state0 : nullptr;
    if (to) {
        const bool across = !PARTS && s.last_t;
        const float f = !PARTS && BACK && sp.n ? power(ld, 1.f) : 1.f;
        each([&](int d, int e, float& v) { to[across ? (long long)e * D + d : (long long)d * E + e] = f * v; });
    }
    if (last_block) wait_for_previous();
}

template <class T, int DP, int EP, bool BACK>
void mma_launch_as(const Scan& s, cudaStream_t st) {
    constexpr int bytes = MmLayout<DP, EP>::floats * 4;
    static OnEachDevice here;
    here.first(current_device(), [] {
        allow_shared(k_decay_mma<T, DP, EP, BACK, false>, bytes);
        allow_shared(k_decay_mma<T, DP, EP, BACK, true>, bytes);
    });
    const auto by4 = [&](const Operand& o) {
        return reinterpret_cast<uintptr_t>(o.p) % (4 * sizeof(T)) == 0 && o.batch % 4 == 0 && o.tick % 4 == 0 && o.head % 4 == 0;
    };
    const int quads = s.D % 4 == 0 && s.E % 4 == 0 && by4(s.a) && by4(s.b) && by4(s.c);
    const unsigned rows = (unsigned)(s.batch * s.heads);
    if (s.parts > 1) k_decay_mma<T, DP, EP, BACK, true><<<dim3(rows, s.parts - 1), kMmThreads, bytes, st>>>(s, quads);
    launch_beside(k_decay_mma<T, DP, EP, BACK, false>, dim3(rows, s.parts), kMmThreads, bytes, st, s, quads);
}
template <class T, bool BACK>
void mma_launch_dims(const Scan& s, cudaStream_t st) {
    if (s.D > 64) s.E > 64 ? mma_launch_as<T, 128, 128, BACK>(s, st) : mma_launch_as<T, 128, 64, BACK>(s, st);
    else s.E > 64 ? mma_launch_as<T, 64, 128, BACK>(s, st) : mma_launch_as<T, 64, 64, BACK>(s, st);
}

}  // namespace
