// The gated delta rule over chunks of 64 ticks. With G the log decays added up from the chunk's first tick on, M_ts = exp(G_t - G_s),
// L = K K^T . M below the diagonal, P = scale Q K^T . M on and below it, B = diag(beta):
//
//   X = (I + L B)^-1 L
//   N = V - e^G K S,  W = N - X B N,  U = B W            W_t = v_t - g_t k_t S_{t-1}, what a tick's key did not foretell
//   O = scale e^G Q S + P U,  S <- e^{G_63} S + (e^{G_63 - G} K)^T U
//
// and back, R the gradient of the state behind the chunk:
//   dU = e^{G_63 - G} K R + P^T dO,  dR = dU - X^T B dU,  dN = B dR = dV,  dbeta = rows of dR . W
//   R <- e^{G_63} R + (scale e^G dO)^T Q - (e^G dN)^T K   (transposed)
//   dlog_decay_t: o_t dO_t - v_t dN_t, added up from the chunk's last tick on, behind which it is <R, S>
//
// k_delta_prep makes X, P and the gates of every chunk, all at once. What is left runs from chunk to chunk, and there each column of the
// state goes its own way: a warp owns 16 of them, S transposed (16 columns x dim) in registers as an accumulator, and every product has
// them for rows: N^T = V^T - S^T K^T, W^T = N^T - (N^T B) X^T, O^T = S^T Q^T + U^T P^T, S^T += U^T K. An accumulator is the next
// product's left operand as it lies, so states, corrections and outputs never leave the registers, and warps meet only to have tiles of
// K, Q, V, X, P loaded (mma.sync: 25% of the tensor cores' rate, but the chain from state to state has no trip through shared
// memory or TMEM in it).
#pragma once
#include "fg_delta.cuh"

namespace {

constexpr int kGates = 5;

struct Delta {
    Operand q, k, v, o, go;
    Operand gq, gk, dn;              // gradients of q, k and v (dN), in T or (gq_f32 ..) fp32
    Gate log_decay, beta, glog_decay, gbeta;
    const float *first, *glast;      // [batch][heads][D][E], or NULL: zeros
    float *last, *gfirst;            // or NULL: not wanted
    const long long* offsets;
    long long batch, ticks, slots;
    int heads, D, E, gq_f32, gk_f32, dn_f32;
    float scale;
    bf16 *x, *p;                     // [slot][head][term][64][64]
    float* gates;                    // [slot][head][5][64]: e^G, e^{G_63 - G}, beta, G as two floats
    uint4 *states, *gstates;         // [slot][head][tile of 16 columns][term][DP / 16][32]: S and R as left operands
    float4* w;                       // [slot][head][tile][8][32]: W^T as accumulators
    char* u;                         // [slot][head][64][16 tiles]: U in bf16 (inputs of one term) or fp32
    float *od, *vdn, *db;            // [slot][head][tile][64]: rows of o dO, v dN, dbeta
    float* anchor;                   // [slot][head][tile]
};

__device__ __forceinline__ Span span_of(const Delta& s, long long b) {
    if (!s.offsets) return {0, s.ticks};
    const long long lo = min(max(s.offsets[b], 0ll), s.ticks), hi = min(max(s.offsets[b + 1], lo), s.ticks);
    return {lo, hi - lo};
}
// the chunks of recording b have the slots from here on; recordings end to end, of n ticks each, take ceil(n / 64) and leave at most one
// slot between them, ticks / 64 + batch in all
__device__ __forceinline__ long long slot_of(const Delta& s, long long b, long long start) {
    return s.offsets ? start / kTicks + b : b * ((s.ticks + kTicks - 1) / kTicks);
}
struct Chunk {
    long long b, first;              // recording, first tick (of the recording's)
    int n;                           // ticks, 0: this slot is empty
};
__device__ __forceinline__ Chunk chunk_of(const Delta& s, long long slot) {
    if (!s.offsets) {
        const long long per = (s.ticks + kTicks - 1) / kTicks, b = slot / per, first = (slot - b * per) * kTicks;
        return {b, first, (int)min((long long)kTicks, s.ticks - first)};
    }
    long long lo = 0, hi = s.batch - 1;                      // the last recording whose slots begin at or before this one
    while (lo < hi) {
        const long long mid = (lo + hi + 1) / 2;
        if (slot_of(s, mid, min(max(s.offsets[mid], 0ll), s.ticks)) <= slot) lo = mid;
        else hi = mid - 1;
    }
    const Span sp = span_of(s, lo);
    const long long first = (slot - slot_of(s, lo, sp.start)) * kTicks;
    return {lo, first, first < 0 ? 0 : (int)max(0ll, min((long long)kTicks, sp.n - first))};
}
template <class T>
__device__ __forceinline__ T* row_of(const Delta& s, const Operand& o, long long b, int h, long long tick) {
    return reinterpret_cast<T*>(o.p) + (s.offsets ? 0 : b * o.batch) + tick * o.tick + (h / o.share) * o.head;
}
__device__ __forceinline__ float* gate_of(const Delta& s, const Gate& o, long long b, int h, long long tick) {
    return o.p + (s.offsets ? 0 : b * o.batch) + tick * o.tick + h * o.head;
}

// ---- X, P and the gates -------------------------------------------------------------------------------------------------

template <class T, int DP>
struct PrepLayout {
    static constexpr int in = Terms<T>::in, kept = Terms<T>::kept, stride = DP + 8, tile = in * kTicks * stride,
                         square = kept * kTicks * kSquare;
    static constexpr int tiles = 2 * tile > 2 * square ? 2 * tile : 2 * square;   // K and Q, later L B and X
    static constexpr int l = kTicks * 68, bytes = 2 * tiles + 4 * (l + 4 * kTicks);
};

// NP: terms of P. A block of 4 warps makes one chunk of one head: warp w the rows 16 w .. of K K^T and Q K^T, then the block (w, w) of X
// by substitution, then X's column block w downwards, X^T as an accumulator like the states of the chain.
template <class T, int DP, int NP>
__global__ void __launch_bounds__(128) k_delta_prep(const __grid_constant__ Delta s) {
    using Lay = PrepLayout<T, DP>;
    constexpr int NI = Lay::in, NS = Lay::kept, kStride = Lay::stride, kPlane = kTicks * kStride, kSq = kTicks * kSquare;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16 *sk = reinterpret_cast<bf16*>(smem), *sq = sk + Lay::tile, *sa = sk, *sx = sk + Lay::square;
    float *sl = reinterpret_cast<float*>(smem + 2 * Lay::tiles), *gh = sl + Lay::l, *gl = gh + kTicks, *beta = gl + kTicks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const long long slot = blockIdx.x;
    const int h = blockIdx.y;
    const Chunk c = chunk_of(s, slot);
    if (c.n == 0) return;
    const long long tick = (s.offsets ? span_of(s, c.b).start : 0) + c.first;
    load_tile<T, NI, DP, kStride, 128>(sk, row_of<const T>(s, s.k, c.b, h, tick), s.k.tick, c.n, s.D, s.k.fast, tid);
    load_tile<T, NI, DP, kStride, 128>(sq, row_of<const T>(s, s.q, c.b, h, tick), s.q.tick, c.n, s.D, s.q.fast, tid);
    async_commit();
    const long long place = slot * s.heads + h;
    if (warp == 0) {
        // Sums of log decays in 64 bits, kept as two floats: a difference of far ones is then as good as a near one's. e^-256 is 0 in
        // fp32, so nothing lower is needed, and minus infinity (a state forgotten) stays out of the differences.
        double sum[2];
        float lv[2], bv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i;
            lv[i] = r < c.n ? *gate_of(s, s.log_decay, c.b, h, tick + r) : 0.f;
            bv[i] = r < c.n ? *gate_of(s, s.beta, c.b, h, tick + r) : 0.f;
            lv[i] = lv[i] < -256.f ? -256.f : lv[i];
        }
        sum[0] = lv[0];
        sum[1] = sum[0] + (double)lv[1];
        double before = sum[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        const double all = __shfl_sync(0xffffffffu, before, 31);
        before -= sum[1];
        float* out = s.gates + place * kGates * kTicks;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i;
            const double v = before + sum[i];
            gh[r] = (float)v;
            gl[r] = (float)(v - (double)gh[r]);
            beta[r] = bv[i];
            out[r] = expf((float)v);
            out[kTicks + r] = expf((float)(all - v));
            out[2 * kTicks + r] = bv[i];
            out[3 * kTicks + r] = gh[r];
            out[4 * kTicks + r] = gl[r];
        }
    }
    async_wait<0>();
    __syncthreads();

    const uint32_t rows_m = at_rows_m(lane, kStride) + smem_at(sk) + 2 * (16 * warp * kStride), rows_n = at_rows_n(lane, kStride) + smem_at(sk);
    const uint32_t to_q = 2 * Lay::tile;
    bf16* p_out = s.p + place * NP * kTicks * kTicks;
    const int r0 = 16 * warp + g;
#pragma unroll 1
    for (int jp = 0; jp <= warp; ++jp) {
        float kk[2][4] = {}, qk[2][4] = {};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            uint32_t a[NI][4], q[NI][4], b[4];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                ldsm(a[i], rows_m + 2 * (i * kPlane + 16 * d));
                ldsm(q[i], rows_m + to_q + 2 * (i * kPlane + 16 * d));
            }
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                ldsm(b, rows_n + 2 * (j * kPlane + 16 * jp * kStride + 16 * d));
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if (i + j >= NS) continue;
                    mma(kk[0], a[i], b[0], b[1]);
                    mma(kk[1], a[i], b[2], b[3]);
                    mma(qk[0], q[i], b[0], b[1]);
                    mma(qk[1], q[i], b[2], b[3]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = r0 + 8 * i, c0 = 16 * jp + 8 * j + 2 * t4;
                float l[2], p[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = expf((gh[t] - gh[c0 + e]) + (gl[t] - gl[c0 + e]));
                    l[e] = t > c0 + e ? kk[j][2 * i + e] * f : 0.f;
                    p[e] = t >= c0 + e ? qk[j][2 * i + e] * (f * s.scale) : 0.f;
                }
                *reinterpret_cast<float2*>(sl + t * 68 + c0) = make_float2(l[0], l[1]);
                uint32_t u[NP];
                terms<NP>(p[0], p[1], u);
#pragma unroll
                for (int n = 0; n < NP; ++n) *reinterpret_cast<uint32_t*>(p_out + (n * kTicks + t) * kTicks + c0) = u[n];
            }
    }
    __syncthreads();                                          // K and Q have been read, L is there

    // L B as terms, blocks on and below the diagonal
    for (int i = tid; i < kTicks * 8; i += 128) {
        const int r = i >> 3, c0 = (i & 7) * 8;
        if (c0 / 16 > r / 16) continue;
        uint32_t u[4][NS];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            terms<NS>(sl[r * 68 + c0 + 2 * j] * beta[c0 + 2 * j], sl[r * 68 + c0 + 2 * j + 1] * beta[c0 + 2 * j + 1], u[j]);
#pragma unroll
        for (int n = 0; n < NS; ++n) *reinterpret_cast<uint4*>(sa + n * kSq + r * kSquare + c0) = make_uint4(u[0][n], u[1][n], u[2][n], u[3][n]);
    }
    // X's block (w, w): lane = column, rows one after another
    if (lane < 16) {
        float y[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const float* row = sl + (16 * warp + t) * 68 + 16 * warp;
            float v = row[lane];
#pragma unroll
            for (int k = 0; k < t; k += 4) {
                const float4 l = *reinterpret_cast<const float4*>(row + k);
                v = fmaf(-l.x, y[k], v);
                if (k + 1 < t) v = fmaf(-l.y, y[k + 1], v);
                if (k + 2 < t) v = fmaf(-l.z, y[k + 2], v);
                if (k + 3 < t) v = fmaf(-l.w, y[k + 3], v);
            }
            y[t] = v * beta[16 * warp + t];
            uint32_t u[NS];
            terms<NS>(v, 0.f, u);
#pragma unroll
            for (int n = 0; n < NS; ++n)
                reinterpret_cast<unsigned short*>(sx)[n * kSq + (16 * warp + t) * kSquare + 16 * warp + lane] = (unsigned short)u[n];
        }
    }
    __syncthreads();
    // X's blocks below it: X_ij = (I - X_ii B) (L_ij - sum_k (L B)_ik X_kj)
    {
        const uint32_t n_at = at_rows_n(lane, kSquare), a_at = smem_at(sa) + n_at, x_at = smem_at(sx) + n_at;
        const int j0 = 16 * warp;
        uint32_t xf[3][NS][4];
#pragma unroll
        for (int n = 0; n < NS; ++n) ldsm_t(xf[0][n], x_at + 2 * (n * kSq + j0 * kSquare + j0));
#pragma unroll
        for (int di = 1; di < 4; ++di) {
            const int i0 = j0 + 16 * di;
            if (i0 >= kTicks) break;
            float acc[2][4] = {};
#pragma unroll
            for (int k = 0; k < di; ++k)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    uint32_t b[4];
                    ldsm(b, a_at + 2 * (j * kSq + i0 * kSquare + j0 + 16 * k));
#pragma unroll
                    for (int i = 0; i + j < NS; ++i) {
                        mma(acc[0], xf[k][i], b[0], b[1]);
                        mma(acc[1], xf[k][i], b[2], b[3]);
                    }
                }
            float y[2][4], by[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = i0 + 8 * j + 2 * t4 + (e & 1);
                    y[j][e] = sl[t * 68 + j0 + g + 8 * (e >> 1)] - acc[j][e];
                    by[j][e] = y[j][e] * -beta[t];
                }
            uint32_t a[NS][4];
            left<NS>(by[0], by[1], a);
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                uint32_t b[4];
                ldsm(b, x_at + 2 * (j * kSq + i0 * kSquare + i0));
#pragma unroll
                for (int i = 0; i + j < NS; ++i) {
                    mma(acc[0], a[i], b[0], b[1]);
                    mma(acc[1], a[i], b[2], b[3]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[j][e] += acc[j][e];
            left<NS>(y[0], y[1], a);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                stsm_t(x_at + 2 * (n * kSq + i0 * kSquare + j0), a[n]);
                if (di < 3) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) xf[di][n][i] = a[n][i];
                }
            }
        }
    }
    __syncthreads();
    bf16* x_out = s.x + place * NS * kTicks * kTicks;
    for (int i = tid; i < NS * kTicks * 8; i += 128)
        if ((i & 7) / 2 <= (i >> 3 & 63) / 16)
            *reinterpret_cast<uint4*>(x_out + i * 8) = *reinterpret_cast<const uint4*>(sx + (i >> 3) * kSquare + (i & 7) * 8);
}

// ---- from chunk to chunk ------------------------------------------------------------------------------------------------

// Tiles of one chunk, in values of bf16
template <class T, int DP, int WARPS, int NP, bool GO>
struct ChainLayout {
    static constexpr int in = Terms<T>::in, kept = Terms<T>::kept, stride = DP + 8, vstride = 16 * WARPS + 8;
    static constexpr int k = 0, q = k + in * kTicks * stride, v = q + in * kTicks * stride, go = v + in * kTicks * vstride,
                         x = go + (GO ? in * kTicks * vstride : 0), p = x + kept * kTicks * kSquare, gates = p + NP * kTicks * kSquare,
                         stage = gates + 3 * kTicks * 2;
    static constexpr int stages = in == 1 ? 2 : 1, bytes = 2 * stage * stages;
    static_assert(bytes <= 227 * 1024, "the tiles fit");
};
template <class T, int DP, int WARPS, int NP, bool GO>
__device__ __forceinline__ void load_chunk(const Delta& s, bf16* to, long long b, int h, long long tick, int n, long long slot, int e0) {
    using Lay = ChainLayout<T, DP, WARPS, NP, GO>;
    constexpr int kThreads = 32 * WARPS;
    const int tid = threadIdx.x;
    const long long place = slot * s.heads + h;
    load_tile<T, Lay::in, DP, Lay::stride, kThreads>(to + Lay::k, row_of<const T>(s, s.k, b, h, tick), s.k.tick, n, s.D, s.k.fast, tid);
    load_tile<T, Lay::in, DP, Lay::stride, kThreads>(to + Lay::q, row_of<const T>(s, s.q, b, h, tick), s.q.tick, n, s.D, s.q.fast, tid);
    load_tile<T, Lay::in, 16 * WARPS, Lay::vstride, kThreads>(to + Lay::v, row_of<const T>(s, s.v, b, h, tick) + e0, s.v.tick, n, s.E - e0,
                                                             s.v.fast, tid);
    if constexpr (GO)
        load_tile<T, Lay::in, 16 * WARPS, Lay::vstride, kThreads>(to + Lay::go, row_of<const T>(s, s.go, b, h, tick) + e0, s.go.tick, n,
                                                                 s.E - e0, s.go.fast, tid);
    load_square<Lay::kept, kThreads>(to + Lay::x, s.x + place * Lay::kept * kTicks * kTicks, tid);
    load_square<NP, kThreads>(to + Lay::p, s.p + place * NP * kTicks * kTicks, tid);
    if (tid < 48) async16(smem_at(to + Lay::gates) + tid * 16, s.gates + place * kGates * kTicks + tid * 4, true);
    async_commit();
}

// The chunks of a recording in turn (from the last one on): f(stage, chunk)
template <class Lay, class Load, class F>
__device__ __forceinline__ void each_chunk(bf16* tiles, int chunks, bool back, Load&& load, F&& f) {
    if (!chunks) return;
    const auto nth = [&](int i) { return back ? chunks - 1 - i : i; };
    if (Lay::stages == 2) load(tiles, nth(0));
#pragma unroll 1
    for (int i = 0; i < chunks; ++i) {
        bf16* now = tiles + (Lay::stages == 2 && (i & 1) ? Lay::stage : 0);
        if (Lay::stages == 1) {
            __syncthreads();                                  // the chunk before has been read
            load(now, nth(i));
        }
        async_wait<0>();
        __syncthreads();
        if (Lay::stages == 2 && i + 1 < chunks) load(tiles + (i & 1 ? 0 : Lay::stage), nth(i + 1));
        f(now, nth(i));
    }
}

// S (or R) transposed between memory [D][E] and a warp's registers: rows e0 + g, e0 + g + 8
template <int DP, class F>
__device__ __forceinline__ void each_value(float (&S)[DP / 8][4], int D, int E, int e0, int lane, F&& f) {
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = e0 + (lane >> 2) + 8 * (i >> 1), d = 8 * j + 2 * (lane & 3) + (i & 1);
            if (d < D && e < E) f((long long)d * E + e, S[j][i]);
        }
}

// A warp's 16 columns of 64 rows, x[j] the transposed accumulators, to `to` (rows `row` values apart) by way of the warp's own columns of
// the planes of a tile that it has read already: n rows, `cols` columns there.
template <class T, int VS>
__device__ __forceinline__ void store_rows(const float (&x)[8][4], bf16* tile, T* to, long long row, int n, int cols, bool fast, int lane) {
    constexpr int kPlane = kTicks * VS, kHalves = sizeof(T) / 2;
    const uint32_t at = smem_at(tile) + at_rows_n(lane, VS);
    __syncwarp();
#pragma unroll
    for (int jp = 0; jp < 4; ++jp) {
        uint32_t r[kHalves][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[2 * jp + (i >> 1)][2 * (i & 1)], b = x[2 * jp + (i >> 1)][2 * (i & 1) + 1];
            if constexpr (sizeof(T) == 4) {                   // upper halves in one plane, lower in another
                r[0][i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                r[1][i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
            } else {
                const T v[2] = {from_f<T>(a), from_f<T>(b)};
                r[0][i] = *reinterpret_cast<const uint32_t*>(v);
            }
        }
#pragma unroll
        for (int k = 0; k < kHalves; ++k) stsm_t(at + 2 * (k * kPlane + 16 * jp * VS), r[k]);
    }
    __syncwarp();
    const int half = lane & 1, c = 8 * half;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = 16 * i + (lane >> 1);
        if (t >= n || c >= cols) continue;
        T* q = to + t * row + c;
        uint4 u[kHalves];
#pragma unroll
        for (int k = 0; k < kHalves; ++k) u[k] = *reinterpret_cast<const uint4*>(tile + k * kPlane + t * VS + c);
        T v[8];
        if constexpr (sizeof(T) == 4) {
            const uint32_t *a = &u[0].x, *b = &u[1].x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = __uint_as_float(__byte_perm(b[k], a[k], 0x5410));
                v[2 * k + 1] = __uint_as_float(__byte_perm(b[k], a[k], 0x7632));
            }
        } else {
            *reinterpret_cast<uint4*>(v) = u[0];
        }
        if (fast) {
#pragma unroll
            for (int k = 0; k < kHalves; ++k) reinterpret_cast<uint4*>(q)[k] = reinterpret_cast<const uint4*>(v)[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k < cols) q[k] = v[k];
        }
    }
    __syncwarp();
}

// x[j] of the warp's columns from NI planes of a tile, transposed as accumulators; j = 2 jp, 2 jp + 1
template <int NI, int VS>
__device__ __forceinline__ void two_columns(uint32_t at, int jp, float (&x)[2][4]) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        uint32_t r[4];
        ldsm_t(r, at + 2 * (n * kTicks * VS + 16 * jp * VS));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float(&v)[4] = x[i >> 1];
            const int c = 2 * (i & 1);
            v[c] = n ? v[c] + low(r[i]) : low(r[i]);
            v[c + 1] = n ? v[c + 1] + high(r[i]) : high(r[i]);
        }
    }
}
// two neighbouring values of a 64-value gate for columns 8 j + 2 t4, + 1
__device__ __forceinline__ float2 gate2(const float* gates, int j, int lane) {
    return *reinterpret_cast<const float2*>(gates + 8 * j + 2 * (lane & 3));
}

// Forward. KEEP: nothing but what the way back needs is written (S before each chunk, W, U, rows of o dO), and o is made to as many
// terms as the states.
template <class T, int DP, int WARPS, bool KEEP>
__global__ void __launch_bounds__(32 * WARPS) k_delta_chain(const __grid_constant__ Delta s) {
    constexpr int NI = Terms<T>::in, NS = Terms<T>::kept, NO = KEEP ? NS : Terms<T>::out;
    using Lay = ChainLayout<T, DP, WARPS, NO, KEEP>;
    constexpr int kPlane = kTicks * Lay::stride, kSq = kTicks * kSquare;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* tiles = reinterpret_cast<bf16*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks_e = (s.E + 16 * WARPS - 1) / (16 * WARPS), tiles_e = (s.E + 15) / 16;
    long long item = blockIdx.x;
    const int e_block = (int)(item % blocks_e) * 16 * WARPS, e0 = e_block + 16 * warp;
    item /= blocks_e;
    const int h = (int)(item % s.heads);
    const long long b = item / s.heads;
    const Span sp = span_of(s, b);
    const int chunks = (int)((sp.n + kTicks - 1) / kTicks);
    const long long slot0 = slot_of(s, b, sp.start), state0 = (b * s.heads + h) * s.D * s.E;
    const bool mine = e0 < s.E;

    float S[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) S[j][0] = S[j][1] = S[j][2] = S[j][3] = 0.f;
    if (s.first) each_value<DP>(S, s.D, s.E, e0, lane, [&](long long at, float& v) { v = s.first[state0 + at]; });

    const auto load = [&](bf16* to, int i) {
        load_chunk<T, DP, WARPS, NO, KEEP>(s, to, b, h, sp.start + (long long)i * kTicks, (int)min((long long)kTicks, sp.n - (long long)i * kTicks),
                                           slot0 + i, e_block);
    };
    each_chunk<Lay>(tiles, chunks, false, load, [&](bf16* now, int i) {
        if (!mine) return;
        const int n = (int)min((long long)kTicks, sp.n - (long long)i * kTicks);
        const long long place = (slot0 + i) * s.heads + h, warp_place = place * tiles_e + e0 / 16;
        const uint32_t rows_n = smem_at(now) + at_rows_n(lane, Lay::stride), rows_m = smem_at(now) + at_rows_m(lane, Lay::stride);
        const uint32_t square_n = smem_at(now) + at_rows_n(lane, kSquare), columns = smem_at(now) + at_rows_k(lane, Lay::vstride) + 32 * warp;
        const float *from0 = reinterpret_cast<const float*>(now + Lay::gates), *to_end = from0 + kTicks, *beta = to_end + kTicks;
        float N[8][4], O[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) N[j][e] = O[j][e] = 0.f;
        // S^T K^T and S^T Q^T
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            uint32_t a[NS][4];
            left<NS>(S[2 * d], S[2 * d + 1], a);
            if constexpr (KEEP) {
#pragma unroll
                for (int k = 0; k < NS; ++k)
                    s.states[((warp_place * NS + k) * (DP / 16) + d) * 32 + lane] = make_uint4(a[k][0], a[k][1], a[k][2], a[k][3]);
            }
#pragma unroll
            for (int jp = 0; jp < 4; ++jp)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    uint32_t r[4];
                    ldsm(r, rows_n + 2 * (Lay::k + j * kPlane + 16 * jp * Lay::stride + 16 * d));
#pragma unroll
                    for (int k = 0; k + j < NS; ++k) {
                        mma(N[2 * jp], a[k], r[0], r[1]);
                        mma(N[2 * jp + 1], a[k], r[2], r[3]);
                    }
                    ldsm(r, rows_n + 2 * (Lay::q + j * kPlane + 16 * jp * Lay::stride + 16 * d));
#pragma unroll
                    for (int k = 0; k + j < NO; ++k) {
                        mma(O[2 * jp], a[k], r[0], r[1]);
                        mma(O[2 * jp + 1], a[k], r[2], r[3]);
                    }
                }
        }
        // N = V - e^G K S; scale e^G Q S
#pragma unroll
        for (int jp = 0; jp < 4; ++jp) {
            float v[2][4];
            two_columns<NI, Lay::vstride>(columns + 2 * Lay::v, jp, v);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f = gate2(from0, 2 * jp + j, lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ge = e & 1 ? f.y : f.x;
                    N[2 * jp + j][e] = fmaf(-ge, N[2 * jp + j][e], v[j][e]);
                    O[2 * jp + j][e] *= ge * s.scale;
                }
            }
        }
        // W = N - X B N
        {
            float Y[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j) Y[j][0] = Y[j][1] = Y[j][2] = Y[j][3] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float x[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 f = gate2(beta, 2 * k + j, lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = N[2 * k + j][e] * (e & 1 ? f.y : f.x);
                }
                uint32_t a[NS][4];
                left<NS>(x[0], x[1], a);
#pragma unroll
                for (int jp = k; jp < 4; ++jp)
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        uint32_t r[4];
                        ldsm(r, square_n + 2 * (Lay::x + j * kSq + 16 * jp * kSquare + 16 * k));
#pragma unroll
                        for (int t = 0; t + j < NS; ++t) {
                            mma(Y[2 * jp], a[t], r[0], r[1]);
                            mma(Y[2 * jp + 1], a[t], r[2], r[3]);
                        }
                    }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) N[j][e] -= Y[j][e];
        }
        if constexpr (KEEP) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s.w[(warp_place * 8 + j) * 32 + lane] = make_float4(N[j][0], N[j][1], N[j][2], N[j][3]);
        }
        // U = B W; O += P U
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = gate2(beta, j, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) N[j][e] *= e & 1 ? f.y : f.x;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t a[NO][4];
            left<NO>(N[2 * k], N[2 * k + 1], a);
#pragma unroll
            for (int jp = k; jp < 4; ++jp)
#pragma unroll
                for (int j = 0; j < NO; ++j) {
                    uint32_t r[4];
                    ldsm(r, square_n + 2 * (Lay::p + j * kSq + 16 * jp * kSquare + 16 * k));
#pragma unroll
                    for (int t = 0; t + j < NO; ++t) {
                        mma(O[2 * jp], a[t], r[0], r[1]);
                        mma(O[2 * jp + 1], a[t], r[2], r[3]);
                    }
                }
        }
        if constexpr (!KEEP) {
            store_rows<T, Lay::vstride>(O, now + Lay::v + 16 * warp, row_of<T>(s, s.o, b, h, sp.start + (long long)i * kTicks) + e0, s.o.tick, n,
                                        s.E - e0, s.o.fast, lane);
        } else {
            float sums[16];
#pragma unroll
            for (int jp = 0; jp < 4; ++jp) {
                float v[2][4];
                two_columns<NI, Lay::vstride>(columns + 2 * Lay::go, jp, v);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) sums[4 * jp + 2 * j + e] = O[2 * jp + j][e] * v[j][e] + O[2 * jp + j][e + 2] * v[j][e + 2];
            }
            const float2 od = column_sums(sums, lane);
            *reinterpret_cast<float2*>(s.od + warp_place * kTicks + 8 * (lane >> 2) + 2 * (lane & 3)) = od;
            using U = std::conditional_t<NI == 1, bf16, float>;
            store_rows<U, Lay::vstride>(N, now + Lay::v + 16 * warp, reinterpret_cast<U*>(s.u) + place * kTicks * 16 * tiles_e + e0,
                                        16 * tiles_e, kTicks, 16, true, lane);
        }
        // S = e^{G_63} S + (e^{G_63 - G} K)^T U
        uint32_t a[4][NS][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float x[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f = gate2(to_end, 2 * k + j, lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = N[2 * k + j][e] * (e & 1 ? f.y : f.x);
            }
            left<NS>(x[0], x[1], a[k]);
        }
        const float fade = from0[kTicks - 1];
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            float acc[2][4] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    uint32_t r[4];
                    ldsm_t(r, rows_m + 2 * (Lay::k + j * kPlane + 16 * k * Lay::stride + 16 * d));
#pragma unroll
                    for (int t = 0; t + j < NS; ++t) {
                        mma(acc[0], a[k][t], r[0], r[1]);
                        mma(acc[1], a[k][t], r[2], r[3]);
                    }
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[2 * d + j][e] = fmaf(S[2 * d + j][e], fade, acc[j][e]);
        }
    });
    if (s.last) each_value<DP>(S, s.D, s.E, e0, lane, [&](long long at, float& v) { s.last[state0 + at] = v; });
}

__device__ __forceinline__ void prefetch(const char* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Back. s.last is the state after the recording's last tick.
template <class T, int DP, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) k_delta_back(const __grid_constant__ Delta s) {
    constexpr int NI = Terms<T>::in, NS = Terms<T>::kept, NG = NI == 1 ? 1 : NS;   // NG: terms of R that the gradients of q and k need
    using Lay = ChainLayout<T, DP, WARPS, NS, true>;
    constexpr int kPlane = kTicks * Lay::stride, kSq = kTicks * kSquare;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* tiles = reinterpret_cast<bf16*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks_e = (s.E + 16 * WARPS - 1) / (16 * WARPS), tiles_e = (s.E + 15) / 16;
    long long item = blockIdx.x;
    const int e_block = (int)(item % blocks_e) * 16 * WARPS, e0 = e_block + 16 * warp;
    item /= blocks_e;
    const int h = (int)(item % s.heads);
    const long long b = item / s.heads;
    const Span sp = span_of(s, b);
    const int chunks = (int)((sp.n + kTicks - 1) / kTicks);
    const long long slot0 = slot_of(s, b, sp.start), state0 = (b * s.heads + h) * s.D * s.E;
    const bool mine = e0 < s.E;

    float R[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) R[j][0] = R[j][1] = R[j][2] = R[j][3] = 0.f;
    if (s.glast) each_value<DP>(R, s.D, s.E, e0, lane, [&](long long at, float& v) { v = s.glast[state0 + at]; });

    const auto load = [&](bf16* to, int i) {
        load_chunk<T, DP, WARPS, NS, true>(s, to, b, h, sp.start + (long long)i * kTicks, (int)min((long long)kTicks, sp.n - (long long)i * kTicks),
                                           slot0 + i, e_block);
    };
    each_chunk<Lay>(tiles, chunks, true, load, [&](bf16* now, int i) {
        if (!mine) return;
        const int n = (int)min((long long)kTicks, sp.n - (long long)i * kTicks);
        const long long place = (slot0 + i) * s.heads + h, warp_place = place * tiles_e + e0 / 16;
        const uint32_t rows_n = smem_at(now) + at_rows_n(lane, Lay::stride), rows_m = smem_at(now) + at_rows_m(lane, Lay::stride);
        const uint32_t square_m = smem_at(now) + at_rows_m(lane, kSquare), columns = smem_at(now) + at_rows_k(lane, Lay::vstride) + 32 * warp;
        const float *from0 = reinterpret_cast<const float*>(now + Lay::gates), *to_end = from0 + kTicks, *beta = to_end + kTicks;
        float N[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) N[j][0] = N[j][1] = N[j][2] = N[j][3] = 0.f;
        // R^T K^T, and <R, S> behind the chunk
        float anchor = 0.f;
        const uint4* behind = s.states + ((place + s.heads) * tiles_e + e0 / 16) * NS * (DP / 16) * 32 + lane;
        const bool inner = i + 1 < chunks;
        uint4 ahead[NS];
        if (inner) {
#pragma unroll
            for (int k = 0; k < NS; ++k) ahead[k] = __ldg(behind + k * (DP / 16) * 32);
        }
        if (i > 0) {                                          // what the next chunk reads of this, on its way to L2
            const char* states = reinterpret_cast<const char*>(s.states + warp_place * NS * (DP / 16) * 32);
            for (int at = lane * 128; at < NS * (DP / 16) * 512; at += 32 * 128) prefetch(states + at);
            prefetch(reinterpret_cast<const char*>(s.w + (warp_place - (long long)s.heads * tiles_e) * 8 * 32) + lane * 128);
        }
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            uint32_t a[NS][4];
            left<NS>(R[2 * d], R[2 * d + 1], a);
#pragma unroll
            for (int k = 0; k < NG; ++k)
                s.gstates[((warp_place * NG + k) * (DP / 16) + d) * 32 + lane] = make_uint4(a[k][0], a[k][1], a[k][2], a[k][3]);
            if (inner) {
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    const uint4 u = ahead[k];
                    if (d + 1 < DP / 16) ahead[k] = __ldg(behind + (k * (DP / 16) + d + 1) * 32);
                    const uint32_t* p = &u.x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float(&v)[4] = R[2 * d + (j >> 1)];
                        anchor = fmaf(v[2 * (j & 1)], low(p[j]), anchor);
                        anchor = fmaf(v[2 * (j & 1) + 1], high(p[j]), anchor);
                    }
                }
            }
#pragma unroll
            for (int jp = 0; jp < 4; ++jp)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    uint32_t r[4];
                    ldsm(r, rows_n + 2 * (Lay::k + j * kPlane + 16 * jp * Lay::stride + 16 * d));
#pragma unroll
                    for (int k = 0; k + j < NS; ++k) {
                        mma(N[2 * jp], a[k], r[0], r[1]);
                        mma(N[2 * jp + 1], a[k], r[2], r[3]);
                    }
                }
        }
        if (i + 1 == chunks) each_value<DP>(R, s.D, s.E, e0, lane, [&](long long at, float& v) { anchor = fmaf(v, s.last[state0 + at], anchor); });
        anchor = warp_sum(anchor);
        if (lane == 0) s.anchor[warp_place] = anchor;
        // dU = e^{G_63 - G} K R + P^T dO
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = gate2(to_end, j, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) N[j][e] *= e & 1 ? f.y : f.x;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t a[NI][4];
#pragma unroll
            for (int t = 0; t < NI; ++t) ldsm_t(a[t], columns + 2 * (Lay::go + t * kTicks * Lay::vstride + 16 * k * Lay::vstride));
#pragma unroll
            for (int jp = 0; jp <= k; ++jp)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    uint32_t r[4];
                    ldsm_t(r, square_m + 2 * (Lay::p + j * kSq + 16 * k * kSquare + 16 * jp));
#pragma unroll
                    for (int t = 0; t < NI && t + j < NS; ++t) {
                        mma(N[2 * jp], a[t], r[0], r[1]);
                        mma(N[2 * jp + 1], a[t], r[2], r[3]);
                    }
                }
        }
        // dR = dU - X^T B dU
        {
            float Y[8][4];
            float4 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __ldg(s.w + (warp_place * 8 + j) * 32 + lane);
#pragma unroll
            for (int j = 0; j < 8; ++j) Y[j][0] = Y[j][1] = Y[j][2] = Y[j][3] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float x[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 f = gate2(beta, 2 * k + j, lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = N[2 * k + j][e] * (e & 1 ? f.y : f.x);
                }
                uint32_t a[NS][4];
                left<NS>(x[0], x[1], a);
#pragma unroll
                for (int jp = 0; jp <= k; ++jp)
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        uint32_t r[4];
                        ldsm_t(r, square_m + 2 * (Lay::x + j * kSq + 16 * k * kSquare + 16 * jp));
#pragma unroll
                        for (int t = 0; t + j < NS; ++t) {
                            mma(Y[2 * jp], a[t], r[0], r[1]);
                            mma(Y[2 * jp + 1], a[t], r[2], r[3]);
                        }
                    }
            }
            float sums[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) N[j][e] -= Y[j][e];
                sums[2 * j] = N[j][0] * w[j].x + N[j][2] * w[j].z;
                sums[2 * j + 1] = N[j][1] * w[j].y + N[j][3] * w[j].w;
            }
            const float2 db = column_sums(sums, lane);
            *reinterpret_cast<float2*>(s.db + warp_place * kTicks + 8 * (lane >> 2) + 2 * (lane & 3)) = db;
            // dN = B dR, rows of v dN
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v[2][4];
                two_columns<NI, Lay::vstride>(columns + 2 * Lay::v, k, v);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 f = gate2(beta, 2 * k + j, lane);
                    float(&x)[4] = N[2 * k + j];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] *= e & 1 ? f.y : f.x;
#pragma unroll
                    for (int e = 0; e < 2; ++e) sums[4 * k + 2 * j + e] = x[e] * v[j][e] + x[e + 2] * v[j][e + 2];
                }
            }
            const float2 vdn = column_sums(sums, lane);
            *reinterpret_cast<float2*>(s.vdn + warp_place * kTicks + 8 * (lane >> 2) + 2 * (lane & 3)) = vdn;
        }
        {
            const long long tick = sp.start + (long long)i * kTicks;
            bf16* room = now + Lay::v + 16 * warp;
            if (sizeof(T) == 2 && !s.dn_f32)
                store_rows<T, Lay::vstride>(N, room, row_of<T>(s, s.dn, b, h, tick) + e0, s.dn.tick, n, s.E - e0, s.dn.fast, lane);
            else if constexpr (NI > 1)
                store_rows<float, Lay::vstride>(N, room, row_of<float>(s, s.dn, b, h, tick) + e0, s.dn.tick, n, s.E - e0, s.dn.fast, lane);
            else {                                            // (one plane: fp32 straight from the registers)
                float* to = row_of<float>(s, s.dn, b, h, tick) + e0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = 8 * j + 2 * (lane & 3) + (e & 1), c = (lane >> 2) + 8 * (e >> 1);
                        if (t < n && e0 + c < s.E) to[t * s.dn.tick + c] = N[j][e];
                    }
            }
        }
        // R = e^{G_63} R + (scale e^G dO)^T Q - (e^G dN)^T K
        const float fade = from0[kTicks - 1];
        uint32_t a[4][NS][4], q[4][NS][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[2][4], x[2][4];
            two_columns<NI, Lay::vstride>(columns + 2 * Lay::go, k, v);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f = gate2(from0, 2 * k + j, lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ge = e & 1 ? f.y : f.x;
                    x[j][e] = N[2 * k + j][e] * -ge;
                    v[j][e] *= ge * s.scale;
                }
            }
            left<NS>(x[0], x[1], a[k]);
            left<NS>(v[0], v[1], q[k]);
        }
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            float acc[2][4] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    uint32_t r[4];
                    ldsm_t(r, rows_m + 2 * (Lay::k + j * kPlane + 16 * k * Lay::stride + 16 * d));
#pragma unroll
                    for (int t = 0; t + j < NS; ++t) {
                        mma(acc[0], a[k][t], r[0], r[1]);
                        mma(acc[1], a[k][t], r[2], r[3]);
                    }
                    ldsm_t(r, rows_m + 2 * (Lay::q + j * kPlane + 16 * k * Lay::stride + 16 * d));
#pragma unroll
                    for (int t = 0; t + j < NS; ++t) {
                        mma(acc[0], q[k][t], r[0], r[1]);
                        mma(acc[1], q[k][t], r[2], r[3]);
                    }
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) R[2 * d + j][e] = fmaf(R[2 * d + j][e], fade, acc[j][e]);
        }
    });
    if (s.gfirst) each_value<DP>(R, s.D, s.E, e0, lane, [&](long long at, float& v) { s.gfirst[state0 + at] = v; });
}

}  // namespace
