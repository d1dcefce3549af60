// The gated delta rule over chunks of 32 ticks. With G the log decays added up from the chunk's first tick on, M_ts = exp(G_t - G_s),
// L = K K^T . M below the diagonal, P = scale Q K^T . M on and below it, B = diag(beta):
//
//   X = (I + L B)^-1 L
//   N = V - e^G K S,  W = N - X B N,  U = B W            W_t = v_t - g_t k_t S_{t-1}, what a tick's key did not foretell
//   O = scale e^G Q S + P U,  S <- e^{G_31} S + (e^{G_31 - G} K)^T U
//
// and back, R the gradient of the state behind the chunk:
//   dU = e^{G_31 - G} K R + P^T dO,  dR = dU - X^T B dU,  dN = B dR = dV,  dbeta = rows of dR . W
//   R <- e^{G_31} R + (scale e^G dO)^T Q - (e^G dN)^T K   (transposed)
//   dlog_decay_t: o_t dO_t - v_t dN_t, added up from a slot's last tick on, behind which it is <R, S>
//
// k_delta_prep makes X, P and the gates of every chunk, all at once. What is left runs from chunk to chunk, and there each column of the
// state goes its own way: a warp owns 16 of them, S transposed (16 columns x dim) in registers as an accumulator, and every product has
// them for rows: N^T = V^T - S^T K^T, W^T = N^T - (N^T B) X^T, O^T = S^T Q^T + U^T P^T, S^T += U^T K. An accumulator is the next
// product's left operand as it lies, so states, corrections and outputs never leave the registers, and warps meet only to have tiles of
// K, Q, V, X, P loaded (mma.sync: 25% of the tensor cores' rate, but the chain from state to state has no trip through shared
// memory or TMEM in it). Chunks of 32 ticks need 16 registers an accumulator of a tick's row where 64 need 32, which leaves room for 12 to
// 16 warps an SM instead of 8.
//
// 64 recordings of 1,024 ticks, 8 heads of 128 in bf16: forward 522 us (310 products a warp and chunk, 301 us of the tensor cores' at 552
// TFLOP/s of mma.sync), with what is kept 800, back 1,015. The tensor pipe is 54%, 49% and 36% busy, issue slots 39%, DRAM 14%, 33% and
// 38%: products of a warp wait for its own splits into terms and the other way round, more than the warps beside it fill; back for S, W and O,
// too. X, P and the gates take 101 us: some 1,700 instructions a warp, of them 100 products.
#pragma once
#include "fg_delta.cuh"

namespace {

constexpr int kGates = 5;

struct Slot {
    long long tick;
    int b, n;
};
struct Delta {
    Operand q, k, v, o, go;
    Operand gq, gk, dn;              // gradients of q, k and v (dN), in T or (gq_f32 ..) fp32
    Operand dn_high, dn_low;         // dN in T of 16 bits as two terms for the gradients of k: of bf16 the first is gv itself
    Gate log_decay, beta, glog_decay, gbeta;
    const float *first, *glast;      // [batch][heads][D][E], or NULL: zeros
    float *last, *kept_last, *gfirst;   // or NULL: not wanted
    const long long* offsets;
    long long batch, ticks, slots;
    int heads, D, E, gq_f32, gk_f32, dn_f32;
    float scale;
    Slot* table;                     // [slot], of recordings end to end
    bf16 *x, *p;                     // [slot][head][chunk][term][32][32]
    float* gates;                    // [slot][head][5][64]: e^G and e^{G_31 - G} of the chunks, beta, G of the slot as two floats
    float4 *states, *gstates;        // [slot][head][tile of 16 columns][DP / 8][32]: S before and R behind, transposed, as accumulators
    float4 *w, *o32;                 // [slot][head][chunk][tile][4][32]: W^T and O^T as accumulators
    float *od, *vdn, *db;            // [slot][head][tile][64]: rows of o dO, v dN, dbeta
    float* anchor;                   // [slot][head][tile]: <R, S> behind
    // few long recordings are split into parts, see k_delta_join
    int parts;
    float *own, *turn, *start;       // [batch][heads][part] of [16 tiles][DP], [DP][DP], [16 tiles][DP], all transposed
};

__device__ __forceinline__ Span span_of(const Delta& s, long long b) {
    if (!s.offsets) return {0, s.ticks};
    const long long lo = min(max(s.offsets[b], 0ll), s.ticks), hi = min(max(s.offsets[b + 1], lo), s.ticks);
    return {lo, hi - lo};
}
// recording b has the slots from here on; recordings end to end, of n ticks each, take ceil(n / 64) and leave at most one
// slot between them, ticks / 64 + batch in all
__device__ __forceinline__ long long slot_of(const Delta& s, long long b, long long start) {
    return s.offsets ? start / kTicks + b : b * ((s.ticks + kTicks - 1) / kTicks);
}
// What a slot holds: n ticks of recording b from `tick` on (of the buffer's, where recordings lie end to end); n = 0: nothing.
__device__ __forceinline__ Slot find_slot(const Delta& s, long long slot) {
    long long lo = 0, hi = s.batch - 1;                      // the last recording whose slots begin at or before this one
    while (lo < hi) {
        const long long mid = (lo + hi + 1) / 2;
        if (slot_of(s, mid, min(max(s.offsets[mid], 0ll), s.ticks)) <= slot) lo = mid;
        else hi = mid - 1;
    }
    const Span sp = span_of(s, lo);
    const long long first = (slot - slot_of(s, lo, sp.start)) * kTicks;
    return {sp.start + first, (int)lo, first < 0 ? 0 : (int)max(0ll, min((long long)kTicks, sp.n - first))};
}
// of packed recordings, once for all blocks that ask (a search is some 8 loads that wait for one another: 97,500 ticks of 130 recordings, 8
// heads, X and P and the gradients of q and k took 908 us with one in each block, now 816)
__global__ void __launch_bounds__(128) k_delta_slots(const __grid_constant__ Delta s) {
    const long long slot = blockIdx.x * 128ll + threadIdx.x;
    if (slot < s.slots) s.table[slot] = find_slot(s, slot);
}
__device__ __forceinline__ Slot ticks_of(const Delta& s, long long slot) {
    if (s.offsets) return s.table[slot];
    const uint32_t per = (uint32_t)((s.ticks + kTicks - 1) / kTicks), b = (uint32_t)slot / per;   // (slots are fewer than 2^31)
    const long long first = (long long)((uint32_t)slot - b * per) * kTicks;
    return {first, (int)b, (int)min((long long)kTicks, s.ticks - first)};
}
// values of a row of dn_high or dn_low
__host__ __device__ constexpr int padded_values(int E) { return (E + 7) / 8 * 8; }
// the chunks of a part: whole slots, as many in each but the last ones
struct Part {
    int first, end;
};
__device__ __forceinline__ Part part_of(const Delta& s, long long n, int part) {
    const long long slots = (n + kTicks - 1) / kTicks, per = 2 * ((slots + s.parts - 1) / s.parts);
    const int chunks = (int)((n + kChunk - 1) / kChunk);
    return {(int)min((long long)chunks, part * per), (int)min((long long)chunks, (part + 1) * per)};
}
template <class T>
__device__ __forceinline__ T* row_of(const Delta& s, const Operand& o, long long b, int h, long long tick) {
    return reinterpret_cast<T*>(o.p) + (s.offsets ? 0 : b * o.batch) + tick * o.tick + (uint32_t)h / (uint32_t)o.share * o.head;
}
__device__ __forceinline__ float* gate_of(const Delta& s, const Gate& o, long long b, int h, long long tick) {
    return o.p + (s.offsets ? 0 : b * o.batch) + tick * o.tick + h * o.head;
}

// ---- X, P and the gates -------------------------------------------------------------------------------------------------

template <class T, int DP>
struct PrepLayout {
    static constexpr int in = Terms<T>::in, square = Terms<T>::kept, stride = DP + 8, tile = in * kTicks * stride,
                         small = 2 * square * kChunk * kSmall;                       // of both chunks
    static constexpr int tiles = 2 * tile > 2 * small ? 2 * tile : 2 * small;        // K and Q, later L B and X
    static constexpr int lrow = kChunk + 4, l = kTicks * lrow, bytes = 2 * tiles + 4 * (l + 3 * kTicks);
};

// NP: terms of P. A block of 4 warps makes one slot of one head: warp w rows 16 w .. of its chunk's K K^T and Q K^T, then its block of X
// on the diagonal by substitution; the block below that by products, X^T as an accumulator like the states of the chain.
template <class T, int DP, int NP>
__global__ void __launch_bounds__(128) k_delta_prep(const __grid_constant__ Delta s) {
    using Lay = PrepLayout<T, DP>;
    constexpr int NI = Lay::in, NX = Lay::square, kStride = Lay::stride, kPlane = kTicks * kStride, kSm = kChunk * kSmall, kL = Lay::lrow;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16 *sk = reinterpret_cast<bf16*>(smem), *sa = sk, *sx = sk + Lay::small;
    float *sl = reinterpret_cast<float*>(smem + 2 * Lay::tiles), *gh = sl + Lay::l, *gl = gh + kTicks, *beta = gl + kTicks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, chunk = warp >> 1, lower = warp & 1;
    const long long slot = blockIdx.x;
    const int h = blockIdx.y;
    const Slot c = ticks_of(s, slot);
    if (c.n == 0) return;
    const long long tick = c.tick;
    load_tile<T, NI, DP, kStride, 128>(sk, row_of<const T>(s, s.k, c.b, h, tick), s.k.tick, c.n, s.D, s.k.fast, tid);
    load_tile<T, NI, DP, kStride, 128>(sk + Lay::tile, row_of<const T>(s, s.q, c.b, h, tick), s.q.tick, c.n, s.D, s.q.fast, tid);
    async_commit();
    const long long place = slot * s.heads + h;
    if (warp == 0) {
        // Sums of log decays in 64 bits, kept as two floats: a difference of far ones is then as good as a near one's. e^-256 is 0 in
        // fp32, so nothing lower is needed, and minus infinity (a state forgotten) stays out of the differences.
        double sum[2];
        float lv[2], bv[2];
        const float *lp = gate_of(s, s.log_decay, c.b, h, tick), *bp = gate_of(s, s.beta, c.b, h, tick);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i;
            lv[i] = r < c.n ? lp[r * s.log_decay.tick] : 0.f;
            bv[i] = r < c.n ? bp[r * s.beta.tick] : 0.f;
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
        const double end = __shfl_sync(0xffffffffu, before, lane | 15), middle = __shfl_sync(0xffffffffu, before, 15);
        before -= sum[1];
        float* out = s.gates + place * kGates * kTicks;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i;
            const double v = before + sum[i];
            gh[r] = (float)v;
            gl[r] = (float)(v - (double)gh[r]);
            beta[r] = bv[i];
            out[r] = expf((float)(lane < 16 ? v : v - middle));
            out[kTicks + r] = expf((float)(end - v));
            out[2 * kTicks + r] = bv[i];
            out[3 * kTicks + r] = gh[r];
            out[4 * kTicks + r] = gl[r];
        }
    }
    async_wait<0>();
    __syncthreads();

    const uint32_t rows_m = at_rows_m(lane, kStride) + smem_at(sk) + 2 * (16 * warp * kStride),
                   rows_n = at_rows_n(lane, kStride) + smem_at(sk) + 2 * (kChunk * chunk * kStride);
    constexpr uint32_t to_q = 2 * Lay::tile;
    bf16* p_out = s.p + (2 * place + chunk) * NP * kChunk * kChunk;
    // the block left of the diagonal (of the lower rows), then the one on it
    float kk[2][2][4] = {}, qk[2][2][4] = {};
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
        uint32_t a[NI][4], q[NI][4], b[4];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            ldsm(a[i], rows_m + 2 * (i * kPlane + 16 * d));
            ldsm(q[i], rows_m + to_q + 2 * (i * kPlane + 16 * d));
        }
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
            if (jp > lower) break;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                ldsm(b, rows_n + 2 * (j * kPlane + 16 * jp * kStride + 16 * d));
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if (i + j >= NX) continue;
                    mma(kk[jp][0], a[i], b[0], b[1]);
                    mma(kk[jp][1], a[i], b[2], b[3]);
                    mma(qk[jp][0], q[i], b[0], b[1]);
                    mma(qk[jp][1], q[i], b[2], b[3]);
                }
            }
        }
    }
    __syncthreads();                                          // K and Q have been read: L B goes over them
    float* l_rows = sl + (kChunk * chunk) * kL;
    bf16 *a_rows = sa + chunk * NX * kSm, *x_rows = sx + chunk * NX * kSm;
    const float *ch = gh + kChunk * chunk, *cl = gl + kChunk * chunk, *cb = beta + kChunk * chunk;
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {
        if (jp > lower) break;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = 16 * lower + g + 8 * i, c0 = 16 * jp + 8 * j + 2 * t4;
                float l[2], p[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = expf((ch[t] - ch[c0 + e]) + (cl[t] - cl[c0 + e]));
                    l[e] = t > c0 + e ? kk[jp][j][2 * i + e] * f : 0.f;
                    p[e] = t >= c0 + e ? qk[jp][j][2 * i + e] * (f * s.scale) : 0.f;
                }
                *reinterpret_cast<float2*>(l_rows + t * kL + c0) = make_float2(l[0], l[1]);
                uint32_t u[NP];
                terms<NP>(p[0], p[1], u);
#pragma unroll
                for (int n = 0; n < NP; ++n) *reinterpret_cast<uint32_t*>(p_out + (n * kChunk + t) * kChunk + c0) = u[n];
                if (jp < lower) {                             // L B left of the diagonal
                    uint32_t v[NX];
                    terms<NX>(l[0] * cb[c0], l[1] * cb[c0 + 1], v);
#pragma unroll
                    for (int n = 0; n < NX; ++n) *reinterpret_cast<uint32_t*>(a_rows + n * kSm + t * kSmall + c0) = v[n];
                }
            }
    }
    __syncwarp();
    // X's block on the diagonal: lane = column, rows one after another
    if (lane < 16) {
        const float* block = l_rows + 16 * lower * (kL + 1);
        const float* b = cb + 16 * lower;
        float y[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const float* row = block + t * kL;
            float v = row[lane];
#pragma unroll
            for (int k = 0; k < t; k += 4) {
                const float4 l = *reinterpret_cast<const float4*>(row + k);
                v = fmaf(-l.x, y[k], v);
                if (k + 1 < t) v = fmaf(-l.y, y[k + 1], v);
                if (k + 2 < t) v = fmaf(-l.z, y[k + 2], v);
                if (k + 3 < t) v = fmaf(-l.w, y[k + 3], v);
            }
            y[t] = v * b[t];
            uint32_t u[NX];
            terms<NX>(v, 0.f, u);
#pragma unroll
            for (int n = 0; n < NX; ++n)
                reinterpret_cast<unsigned short*>(x_rows)[n * kSm + (16 * lower + t) * kSmall + 16 * lower + lane] = (unsigned short)u[n];
        }
    }
    __syncthreads();
    // the block below: X_10 = (I - X_11 B) (L_10 - (L B)_10 X_00)
    if (!lower) {
        const uint32_t n_at = at_rows_n(lane, kSmall), a_at = smem_at(a_rows) + n_at, x_at = smem_at(x_rows) + n_at;
        uint32_t x[NX][4];
        float acc[2][4] = {}, y[2][4], by[2][4];
#pragma unroll
        for (int n = 0; n < NX; ++n) ldsm_t(x[n], x_at + 2 * (n * kSm));
        const auto products = [&](uint32_t at) {
#pragma unroll
            for (int j = 0; j < NX; ++j) {
                uint32_t b[4];
                ldsm(b, at + 2 * (j * kSm));
#pragma unroll
                for (int i = 0; i + j < NX; ++i) {
                    mma(acc[0], x[i], b[0], b[1]);
                    mma(acc[1], x[i], b[2], b[3]);
                }
            }
        };
        products(a_at + 2 * (16 * kSmall));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = 16 + 8 * j + 2 * t4 + (e & 1);
                y[j][e] = l_rows[t * kL + g + 8 * (e >> 1)] - acc[j][e];
                by[j][e] = y[j][e] * -cb[t];
                acc[j][e] = 0.f;
            }
        left<NX>(by[0], by[1], x);
        products(x_at + 2 * (16 * kSmall + 16));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[j][e] += acc[j][e];
        left<NX>(y[0], y[1], x);
#pragma unroll
        for (int n = 0; n < NX; ++n) stsm_t(x_at + 2 * (n * kSm + 16 * kSmall), x[n]);
    }
    __syncthreads();
    bf16* x_out = s.x + 2 * place * NX * kChunk * kChunk;
    for (int i = tid; i < 2 * NX * kChunk * 4; i += 128)
        if ((i & 3) / 2 <= (i >> 2 & 31) / 16)
            *reinterpret_cast<uint4*>(x_out + i * 8) = *reinterpret_cast<const uint4*>(sx + (i >> 2) * kSmall + (i & 3) * 8);
}

// ---- from chunk to chunk ------------------------------------------------------------------------------------------------

// Tiles of one chunk, in values of bf16
template <class T, int DP, int WARPS, int NP, bool GO>
struct ChainLayout {
    static constexpr int in = Terms<T>::in, square = Terms<T>::kept, stride = DP + 8, vstride = 16 * WARPS + 8;
    static constexpr int k = 0, q = k + in * kChunk * stride, v = q + in * kChunk * stride, go = v + in * kChunk * vstride,
                         x = go + (GO ? in * kChunk * vstride : 0), p = x + square * kChunk * kSmall, gates = p + NP * kChunk * kSmall,
                         stage = gates + 3 * kChunk * 2;
    static constexpr int stages = in == 1 ? 2 : 1, bytes = 2 * stage * stages;
    static_assert(bytes <= 227 * 1024, "the tiles fit");
};
// What a block reads and writes of its recording and head
template <class T>
struct Source {
    const T *k, *q, *v, *go;
    long long place;                 // of its first slot, in slots times heads
};
template <class T, int DP, int WARPS, int NP, bool GO, bool Q = true>
__device__ __forceinline__ void load_chunk(const Delta& s, const Source<T>& from, bf16* to, int i, int n, int cols) {
    using Lay = ChainLayout<T, DP, WARPS, NP, GO>;
    constexpr int kThreads = 32 * WARPS, kTile = kChunk * kChunk;
    const int tid = threadIdx.x;
    const long long t = (long long)i * kChunk, place = from.place + (long long)(i >> 1) * s.heads, half = 2 * place + (i & 1);
    load_tile<T, Lay::in, DP, Lay::stride, kThreads, kChunk>(to + Lay::k, from.k + t * s.k.tick, s.k.tick, n, s.D, s.k.fast, tid);
    load_tile<T, Lay::in, 16 * WARPS, Lay::vstride, kThreads, kChunk>(to + Lay::v, from.v + t * s.v.tick, s.v.tick, n, cols, s.v.fast, tid);
    load_small<Lay::square, kThreads>(to + Lay::x, s.x + half * Lay::square * kTile, tid);
    if (tid < 24) {
        const int row = tid >> 3, c = (tid & 7) * 4;
        async16(smem_at(to + Lay::gates) + tid * 16, s.gates + (place * kGates + row) * kTicks + (i & 1) * kChunk + c, true);
    }
    if constexpr (Q) load_tile<T, Lay::in, DP, Lay::stride, kThreads, kChunk>(to + Lay::q, from.q + t * s.q.tick, s.q.tick, n, s.D, s.q.fast, tid);
    if constexpr (GO)
        load_tile<T, Lay::in, 16 * WARPS, Lay::vstride, kThreads, kChunk>(to + Lay::go, from.go + t * s.go.tick, s.go.tick, n, cols, s.go.fast, tid);
    if constexpr (Q) load_small<NP, kThreads>(to + Lay::p, s.p + half * NP * kTile, tid);
    async_commit();
}

// The chunks of a part in turn (from the last one on): f(stage, chunk)
template <class Lay, class Load, class F>
__device__ __forceinline__ void each_chunk(bf16* tiles, Part part, bool back, Load&& load, F&& f) {
    const int chunks = part.end - part.first;
    if (!chunks) return;
    const auto nth = [&](int i) { return back ? part.end - 1 - i : part.first + i; };
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

__device__ __forceinline__ void clear(float (&x)[4]) { x[0] = x[1] = x[2] = x[3] = 0.f; }
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

// the same of a part's rows [16 tiles][DP]
template <int DP, class F>
__device__ __forceinline__ void each_pair(float (&S)[DP / 8][4], int e0, int lane, F&& f) {
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) f((e0 + (lane >> 2) + 8 * i) * DP + 8 * j + 2 * (lane & 3), S[j][2 * i], S[j][2 * i + 1]);
}

// A warp's 16 columns of 32 rows, x[j] the transposed accumulators, to `to` (rows `row` values apart) by way of the warp's own columns of
// the planes of a tile that it has read already: n rows, `cols` columns there.
template <class T, int VS>
__device__ __forceinline__ void store_rows(const float (&x)[4][4], bf16* tile, T* to, long long row, int n, int cols, bool fast, int lane) {
    constexpr int kPlane = kChunk * VS, kHalves = sizeof(T) / 2;
    const uint32_t at = smem_at(tile) + at_rows_n(lane, VS);
    __syncwarp();
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {
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
    const int c = 8 * (lane & 1);
    T* q = to + (lane >> 1) * row + c;
#pragma unroll
    for (int i = 0; i < 2; ++i, q += 16 * row) {
        const int t = 16 * i + (lane >> 1);
        if (t >= n || c >= cols) continue;
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

// the warp's columns of 16 ticks from NI planes of a tile, transposed as two accumulators
template <int NI, int VS>
__device__ __forceinline__ void two_columns(uint32_t at, int jp, float (&x)[2][4]) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        uint32_t r[4];
        ldsm_t(r, at + 2 * (n * kChunk * VS + 16 * jp * VS));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float(&v)[4] = x[i >> 1];
            const int c = 2 * (i & 1);
            v[c] = n ? v[c] + low(r[i]) : low(r[i]);
            v[c + 1] = n ? v[c + 1] + high(r[i]) : high(r[i]);
        }
    }
}
// two neighbouring values of a gate for columns 8 j + 2 t4, + 1
__device__ __forceinline__ float2 gate2(const float* gates, int j, int lane) {
    return *reinterpret_cast<const float2*>(gates + 8 * j + 2 * (lane & 3));
}
__device__ __forceinline__ void scale2(float (&x)[4], float2 f) {
    x[0] *= f.x, x[1] *= f.y, x[2] *= f.x, x[3] *= f.y;
}
// x = x f + y
__device__ __forceinline__ void scale_add(float (&x)[4], float2 f, const float (&y)[4]) {
    x[0] = fmaf(x[0], f.x, y[0]), x[1] = fmaf(x[1], f.y, y[1]), x[2] = fmaf(x[2], f.x, y[2]), x[3] = fmaf(x[3], f.y, y[3]);
}
__device__ __forceinline__ void subtract(float (&x)[4], const float (&y)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] -= y[e];
}

// Blocks of an SM at once: 16 warps with 128 registers a thread as blocks of 8 warps, 12 with 168 as blocks of 4 (at dim 64, 97,500 ticks, 8
// heads: with what is kept and back 441 and 523 us; before O was kept 478 and 508, with 16 warps 595 and 557).
constexpr int chain_blocks(int warps) { return warps == 8 ? 2 : 3; }

// Forward. kKeep: what the way back needs is written, too (S before each slot, W, O in fp32), o (if wanted) is made to as many
// terms as the corrections. kParts: what a part makes of a state of zeros, and (tiles past those of the columns) of the columns of 1.
enum { kForward, kKeep, kParts };
template <class T, int DP, int WARPS, int MODE>
__global__ void __launch_bounds__(32 * WARPS, Terms<T>::in == 1 ? chain_blocks(WARPS) : DP > 64 ? 2 : 3)
    k_delta_chain(const __grid_constant__ Delta s) {
    constexpr bool KEEP = MODE == kKeep, PARTS = MODE == kParts;
    constexpr int NI = Terms<T>::in, NX = Terms<T>::kept, NS = NX, NO = KEEP ? NX : Terms<T>::out_s, NP = KEEP ? NX : Terms<T>::out_p;
    // Q S beside K S, S's terms made once, or after W, with 16 fewer registers held: with what is kept and 128 registers 800 and 1,083 us (64
    // recordings of 1,024 ticks, 8 heads of 128), forward with 168 504 and 501 (P of one term; 522 with two), with what is kept at dim 64 497 and 441
    constexpr bool kTogether = WARPS == 8;
    using Lay = ChainLayout<T, DP, WARPS, NP, false>;
    constexpr int kPlane = kChunk * Lay::stride, kSm = kChunk * kSmall;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* tiles = reinterpret_cast<bf16*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_e = (s.E + 15) / 16, all_tiles = tiles_e + (PARTS ? (s.D + 15) / 16 : 0), blocks_e = (all_tiles + WARPS - 1) / WARPS;
    long long item = blockIdx.x;
    const int e_block = (int)(item % blocks_e) * 16 * WARPS, e0 = e_block + 16 * warp;
    item /= blocks_e;
    const int h = (int)(item % s.heads);
    const long long b = item / s.heads;
    const Span sp = span_of(s, b);
    const int chunks = (int)((sp.n + kChunk - 1) / kChunk);
    const Part part = part_of(s, sp.n, blockIdx.y);
    const long long part_place = (b * s.heads + h) * s.parts + blockIdx.y;
    const long long state0 = (b * s.heads + h) * s.D * s.E;
    const bool mine = e0 < 16 * all_tiles;
    const Source<T> from{row_of<const T>(s, s.k, b, h, sp.start), row_of<const T>(s, s.q, b, h, sp.start),
                         row_of<const T>(s, s.v, b, h, sp.start) + e_block, nullptr, slot_of(s, b, sp.start) * s.heads + h};
    T* out = MODE == kForward || (KEEP && s.o.p) ? row_of<T>(s, s.o, b, h, sp.start) + e0 : nullptr;
    const auto ticks = [&](int i) { return (int)min((long long)kChunk, sp.n - (long long)i * kChunk); };

    float S[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) clear(S[j]);
    if constexpr (PARTS) {
        const int one = e0 - 16 * tiles_e + (lane >> 2) - 2 * (lane & 3);   // the value d = row, counted from the thread's first
        if (e0 >= 16 * tiles_e) {
#pragma unroll
            for (int j = 0; j < DP / 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[j][i] = 8 * j + (i & 1) == one + 8 * (i >> 1) ? 1.f : 0.f;
        }
    } else if (blockIdx.y) {
        if (mine) {
            const float* from = s.start + part_place * 16 * tiles_e * DP;
            each_pair<DP>(S, e0, lane, [&](int at, float& x, float& y) {
                const float2 v = *reinterpret_cast<const float2*>(from + at);
                x = v.x, y = v.y;
            });
        }
    } else if (s.first) {
        each_value<DP>(S, s.D, s.E, e0, lane, [&](long long at, float& v) { v = s.first[state0 + at]; });
    }

    const auto load = [&](bf16* to, int i) { load_chunk<T, DP, WARPS, NP, false, !PARTS>(s, from, to, i, ticks(i), s.E - e_block); };
    each_chunk<Lay>(tiles, part, false, load, [&](bf16* now, int i) {
        if (!mine) return;
        const uint32_t tile = smem_at(now), rows_n = tile + at_rows_n(lane, Lay::stride), rows_m = tile + at_rows_m(lane, Lay::stride),
                       square_n = tile + at_rows_n(lane, kSmall), columns = tile + at_rows_k(lane, Lay::vstride) + 32 * warp;
        const float *from0 = reinterpret_cast<const float*>(now + Lay::gates), *to_end = from0 + kChunk, *beta = to_end + kChunk;
        const long long place = from.place + (long long)(i >> 1) * s.heads, warp_place = place * tiles_e + e0 / 16;
        float N[4][4], O[4][4];
        const auto query = [&](const auto& a, int d) {
            products<sizeof(a) / 16, NI, NO, 2, false>(O, a, [&](int j, int p) { return rows_n + 2 * (Lay::q + j * kPlane + 16 * p * Lay::stride + 16 * d); },
                                                       d == 0);
        };
        // N = V - e^G K S
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            uint32_t a[NS][4];
            left<NS>(S[2 * d], S[2 * d + 1], a);
            if (KEEP && !(i & 1)) {
#pragma unroll
                for (int j = 2 * d; j < 2 * d + 2; ++j)
                    s.states[(warp_place * (DP / 8) + j) * 32 + lane] = make_float4(S[j][0], S[j][1], S[j][2], S[j][3]);
            }
            products<NS, NI, NS, 2, false>(N, a, [&](int j, int p) { return rows_n + 2 * (Lay::k + j * kPlane + 16 * p * Lay::stride + 16 * d); }, d == 0);
            if (kTogether && !PARTS) query(a, d);
        }
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
            float v[2][4];
            two_columns<NI, Lay::vstride>(columns + 2 * Lay::v, jp, v);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f = gate2(from0, 2 * jp + j, lane);
                scale_add(N[2 * jp + j], make_float2(-f.x, -f.y), v[j]);
            }
        }
        // W = N - X B N; U = B W
        {
            float Y[4][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float x[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = N[2 * k + j][e];
                    scale2(x[j], gate2(beta, 2 * k + j, lane));
                }
                uint32_t a[NX][4];
                left<NX>(x[0], x[1], a);
                const auto at = [&](int j, int p) { return square_n + 2 * (Lay::x + j * kSm + 16 * (p + k) * kSmall + 16 * k); };
                if (k == 0) products<NX, NX, NX, 2, false>(Y, a, at, true);
                else products<NX, NX, NX, 1, false>(Y + 2, a, at);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) subtract(N[j], Y[j]);
        }
        const long long w_place = (2 * place + (i & 1)) * tiles_e + e0 / 16;
        if constexpr (KEEP) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s.w[(w_place * 4 + j) * 32 + lane] = make_float4(N[j][0], N[j][1], N[j][2], N[j][3]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) scale2(N[j], gate2(beta, j, lane));
        // O = scale e^G Q S + P U
        if constexpr (!PARTS) {
            if (!kTogether) {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t a[NO][4];
                    left<NO>(S[2 * d], S[2 * d + 1], a);
                    query(a, d);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = gate2(from0, j, lane);
                scale2(O[j], make_float2(f.x * s.scale, f.y * s.scale));
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t a[NP][4];
                left<NP>(N[2 * k], N[2 * k + 1], a);
                const auto at = [&](int j, int p) { return square_n + 2 * (Lay::p + j * kSm + 16 * (p + k) * kSmall + 16 * k); };
                if (k == 0) products<NP, NP, NP, 2, false>(O, a, at);
                else products<NP, NP, NP, 1, false>(O + 2, a, at);
            }
            if constexpr (KEEP) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s.o32[(w_place * 4 + j) * 32 + lane] = make_float4(O[j][0], O[j][1], O[j][2], O[j][3]);
            }
            if (!KEEP || out)
                store_rows<T, Lay::vstride>(O, now + Lay::v + 16 * warp, out + (long long)i * kChunk * s.o.tick, s.o.tick, ticks(i), s.E - e0, s.o.fast, lane);
        }
        // S = e^{G_31} S + (e^{G_31 - G} K)^T U
        uint32_t a[2][NS][4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int j = 0; j < 2; ++j) scale2(N[2 * k + j], gate2(to_end, 2 * k + j, lane));
            left<NS>(N[2 * k], N[2 * k + 1], a[k]);
        }
        const float fade = from0[kChunk - 1];
#pragma unroll
        for (int d = 0; d < DP / 16; d += 2) {
            float acc[4][4];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                products<NS, NI, NS, 2, true>(acc, a[k], [&](int j, int p) { return rows_m + 2 * (Lay::k + j * kPlane + 16 * k * Lay::stride + 16 * (d + p)); }, k == 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) scale_add(S[2 * d + j], make_float2(fade, fade), acc[j]);
        }
    });
    if constexpr (PARTS) {
        if (!mine) return;
        const bool turn = e0 >= 16 * tiles_e;
        float* to = turn ? s.turn + part_place * DP * DP : s.own + part_place * 16 * tiles_e * DP;
        each_pair<DP>(S, turn ? e0 - 16 * tiles_e : e0, lane, [&](int at, float& x, float& y) { *reinterpret_cast<float2*>(to + at) = make_float2(x, y); });
    } else if (chunks ? part.first < chunks && part.end == chunks : blockIdx.y == 0) {
        if (s.last) each_value<DP>(S, s.D, s.E, e0, lane, [&](long long at, float& v) { s.last[state0 + at] = v; });
        if (KEEP) each_value<DP>(S, s.D, s.E, e0, lane, [&](long long at, float& v) { s.kept_last[state0 + at] = v; });
    }
}

__device__ __forceinline__ void prefetch(const char* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Back. s.kept_last is the state after the recording's last tick. PARTS: what a part leaves of a gradient of zeros, and nothing else.
template <class T, int DP, int WARPS, bool PARTS>
__global__ void __launch_bounds__(32 * WARPS, Terms<T>::in == 1 ? chain_blocks(WARPS) : DP > 64 ? 2 : 3)
    k_delta_back(const __grid_constant__ Delta s) {
    constexpr int NI = Terms<T>::in, NX = Terms<T>::kept, NS = NX;
    using Lay = ChainLayout<T, DP, WARPS, NX, true>;
    constexpr bool kEarly = DP == 64;
    constexpr int kPlane = kChunk * Lay::stride, kSm = kChunk * kSmall;
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
    const int chunks = (int)((sp.n + kChunk - 1) / kChunk);
    const Part part = part_of(s, sp.n, blockIdx.y);
    const long long part_place = (b * s.heads + h) * s.parts + blockIdx.y;
    const long long state0 = (b * s.heads + h) * s.D * s.E;
    const bool mine = e0 < s.E;
    const Source<T> from{row_of<const T>(s, s.k, b, h, sp.start), row_of<const T>(s, s.q, b, h, sp.start),
                         row_of<const T>(s, s.v, b, h, sp.start) + e_block, row_of<const T>(s, s.go, b, h, sp.start) + e_block,
                         slot_of(s, b, sp.start) * s.heads + h};
    const auto ticks = [&](int i) { return (int)min((long long)kChunk, sp.n - (long long)i * kChunk); };

    float R[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) clear(R[j]);
    if (PARTS) {
    } else if ((int)blockIdx.y + 1 < s.parts) {
        if (mine) {
            const float* at_end = s.start + part_place * 16 * tiles_e * DP;
            each_pair<DP>(R, e0, lane, [&](int at, float& x, float& y) {
                const float2 v = *reinterpret_cast<const float2*>(at_end + at);
                x = v.x, y = v.y;
            });
        }
    } else if (s.glast) {
        each_value<DP>(R, s.D, s.E, e0, lane, [&](long long at, float& v) { v = s.glast[state0 + at]; });
    }
    if (!PARTS && mine && (chunks & 1) && part.first < chunks && part.end == chunks) {   // a slot's second chunk without ticks
        const long long at = ((from.place + (long long)(chunks >> 1) * s.heads) * tiles_e + e0 / 16) * kTicks + kChunk + lane;
        s.od[at] = s.vdn[at] = s.db[at] = 0.f;
    }

    const auto load = [&](bf16* to, int i) { load_chunk<T, DP, WARPS, NX, true>(s, from, to, i, ticks(i), s.E - e_block); };
    each_chunk<Lay>(tiles, part, true, load, [&](bf16* now, int i) {
        if (!mine) return;
        const uint32_t tile = smem_at(now), rows_n = tile + at_rows_n(lane, Lay::stride), rows_m = tile + at_rows_m(lane, Lay::stride),
                       square_m = tile + at_rows_m(lane, kSmall), columns = tile + at_rows_k(lane, Lay::vstride) + 32 * warp;
        const float *from0 = reinterpret_cast<const float*>(now + Lay::gates), *to_end = from0 + kChunk, *beta = to_end + kChunk;
        const long long place = from.place + (long long)(i >> 1) * s.heads, warp_place = place * tiles_e + e0 / 16;
        const long long w_place = (2 * place + (i & 1)) * tiles_e + e0 / 16;
        const bool last = i + 1 == chunks, slot_end = !PARTS && ((i & 1) || last);   // R is the one behind the slot
        const float4* behind = s.states + (warp_place + (long long)s.heads * tiles_e) * (DP / 8) * 32 + lane;
        if (!PARTS && i > part.first) {                       // what the next chunk reads of this, on its way to L2
            if (!(i & 1)) {
                const char* states = reinterpret_cast<const char*>(s.states + warp_place * (DP / 8) * 32);
                for (int at = lane * 128; at < DP / 8 * 512; at += 32 * 128) prefetch(states + at);
            }
            const long long before = (2 * (place - (i & 1 ? 0 : s.heads)) + !(i & 1)) * tiles_e + e0 / 16;
            prefetch(reinterpret_cast<const char*>((lane < 16 ? s.w : s.o32) + before * 4 * 32) + (lane & 15) * 128);
        }
        float N[4][4];
        // R^T K^T, and <R, S> behind the slot
        float anchor = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            float4 kept[2];
            if (slot_end && !last) {
#pragma unroll
                for (int j = 0; j < 2; ++j) kept[j] = __ldg(behind + (2 * d + j) * 32);
            }
            if (slot_end) {
#pragma unroll
                for (int j = 2 * d; j < 2 * d + 2; ++j)
                    s.gstates[(warp_place * (DP / 8) + j) * 32 + lane] = make_float4(R[j][0], R[j][1], R[j][2], R[j][3]);
            }
            uint32_t a[NS][4];
            left<NS>(R[2 * d], R[2 * d + 1], a);
            products<NS, NI, NS, 2, false>(N, a, [&](int j, int p) { return rows_n + 2 * (Lay::k + j * kPlane + 16 * p * Lay::stride + 16 * d); }, d == 0);
            if (slot_end && !last) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float(&v)[4] = R[2 * d + j];
                    anchor = fmaf(v[0], kept[j].x, fmaf(v[1], kept[j].y, fmaf(v[2], kept[j].z, fmaf(v[3], kept[j].w, anchor))));
                }
            }
        }
        if (last && !PARTS) each_value<DP>(R, s.D, s.E, e0, lane, [&](long long at, float& v) { anchor = fmaf(v, s.kept_last[state0 + at], anchor); });
        if (slot_end) {
            anchor = warp_sum(anchor);
            if (lane == 0) s.anchor[warp_place] = anchor;
        }
        // dU = e^{G_31 - G} K R + P^T dO
#pragma unroll
        for (int j = 0; j < 4; ++j) scale2(N[j], gate2(to_end, j, lane));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t a[NI][4];
#pragma unroll
            for (int t = 0; t < NI; ++t) ldsm_t(a[t], columns + 2 * (Lay::go + t * kChunk * Lay::vstride + 16 * k * Lay::vstride));
            const auto at = [&](int j, int p) { return square_m + 2 * (Lay::p + j * kSm + 16 * k * kSmall + 16 * p); };
            if (k == 0) products<NI, NX, NX, 1, true>(N, a, at);
            else products<NI, NX, NX, 2, true>(N, a, at);
        }
        // dR = dU - X^T B dU
        const int column = (i & 1) * kChunk + 8 * (lane >> 3) + 2 * (lane & 3) + (lane >> 2 & 1);
        float4 o[4];                                          // (asked for where registers are free)
        const auto fetch_o = [&]() {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __ldg(s.o32 + (w_place * 4 + j) * 32 + lane);
        };
        if (!PARTS && kEarly) fetch_o();
        {
            float Y[4][4];
            float4 w[4];
            if constexpr (!PARTS) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = __ldg(s.w + (w_place * 4 + j) * 32 + lane);
            }
#pragma unroll
            for (int k = 1; k >= 0; --k) {
                float x[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = N[2 * k + j][e];
                    scale2(x[j], gate2(beta, 2 * k + j, lane));
                }
                uint32_t a[NX][4];
                left<NX>(x[0], x[1], a);
                const auto at = [&](int j, int p) { return square_m + 2 * (Lay::x + j * kSm + 16 * k * kSmall + 16 * p); };
                if (k == 0) products<NX, NX, NX, 1, true>(Y, a, at);
                else products<NX, NX, NX, 2, true>(Y, a, at, true);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) subtract(N[j], Y[j]);
            // dN = B dR; rows of dR W and of v dN
            float sums[8];
            if constexpr (!PARTS) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sums[2 * j] = N[j][0] * w[j].x + N[j][2] * w[j].z;
                    sums[2 * j + 1] = N[j][1] * w[j].y + N[j][3] * w[j].w;
                }
                s.db[warp_place * kTicks + column] = column_sums(sums, lane);
                if (!kEarly) fetch_o();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) scale2(N[j], gate2(beta, j, lane));
            if constexpr (!PARTS) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float v[2][4];
                    two_columns<NI, Lay::vstride>(columns + 2 * Lay::v, k, v);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            sums[4 * k + 2 * j + e] = N[2 * k + j][e] * v[j][e] + N[2 * k + j][e + 2] * v[j][e + 2];
                }
                s.vdn[warp_place * kTicks + column] = column_sums(sums, lane);
            }
        }
        if constexpr (!PARTS) {
            const long long tick = sp.start + (long long)i * kChunk;
            const int n = ticks(i);
            bf16* room = now + Lay::v + 16 * warp;
            if (sizeof(T) == 2 && !s.dn_f32) {
                store_rows<T, Lay::vstride>(N, room, row_of<T>(s, s.dn, b, h, tick) + e0, s.dn.tick, n, s.E - e0, s.dn.fast, lane);
                const int whole = padded_values(s.E) - e0;    // (columns past E are zeros)
                if constexpr (!std::is_same<T, bf16>::value)
                    store_rows<bf16, Lay::vstride>(N, room, row_of<bf16>(s, s.dn_high, b, h, tick) + e0, s.dn_high.tick, n, whole, true, lane);
                float rest[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) rest[j][e] = N[j][e] - to_f(from_f<bf16>(N[j][e]));
                store_rows<bf16, Lay::vstride>(rest, room, row_of<bf16>(s, s.dn_low, b, h, tick) + e0, s.dn_low.tick, n, whole, true, lane);
            } else if constexpr (NI > 1)
                store_rows<float, Lay::vstride>(N, room, row_of<float>(s, s.dn, b, h, tick) + e0, s.dn.tick, n, s.E - e0, s.dn.fast, lane);
            else {                                            // (one plane: fp32 straight from the registers)
                float* to = row_of<float>(s, s.dn, b, h, tick) + e0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = 8 * j + 2 * (lane & 3) + (e & 1), c = (lane >> 2) + 8 * (e >> 1);
                        if (t < n && e0 + c < s.E) to[t * s.dn.tick + c] = N[j][e];
                    }
            }
        }
        // R = e^{G_31} R + (scale e^G dO)^T Q - (e^G dN)^T K
        const float fade = from0[kChunk - 1];
        uint32_t a[2][NS][4], q[2][NX][4];
        float dots[8];                                        // rows of o dO
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v[2][4];
            two_columns<NI, Lay::vstride>(columns + 2 * Lay::go, k, v);
            if constexpr (!PARTS) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    dots[4 * k + 2 * j] = fmaf(o[2 * k + j].x, v[j][0], o[2 * k + j].z * v[j][2]);
                    dots[4 * k + 2 * j + 1] = fmaf(o[2 * k + j].y, v[j][1], o[2 * k + j].w * v[j][3]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f = gate2(from0, 2 * k + j, lane);
                scale2(N[2 * k + j], make_float2(-f.x, -f.y));
                scale2(v[j], make_float2(f.x * s.scale, f.y * s.scale));
            }
            left<NS>(N[2 * k], N[2 * k + 1], a[k]);
            left<NX>(v[0], v[1], q[k]);
        }
        if constexpr (!PARTS) s.od[warp_place * kTicks + column] = column_sums(dots, lane);
#pragma unroll
        for (int d = 0; d < DP / 16; d += 2) {
            float acc[4][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                products<NS, NI, NS, 2, true>(acc, a[k], [&](int j, int p) { return rows_m + 2 * (Lay::k + j * kPlane + 16 * k * Lay::stride + 16 * (d + p)); }, k == 0);
                products<NX, NI, NX, 2, true>(acc, q[k], [&](int j, int p) { return rows_m + 2 * (Lay::q + j * kPlane + 16 * k * Lay::stride + 16 * (d + p)); });
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) scale_add(R[2 * d + j], make_float2(fade, fade), acc[j]);
        }
    });
    if constexpr (PARTS) {
        float* to = s.own + part_place * 16 * tiles_e * DP;
        if (mine) each_pair<DP>(R, e0, lane, [&](int at, float& x, float& y) { *reinterpret_cast<float2*>(to + at) = make_float2(x, y); });
    } else if (s.gfirst && blockIdx.y == 0) {
        each_value<DP>(R, s.D, s.E, e0, lane, [&](long long at, float& v) { s.gfirst[state0 + at] = v; });
    }
}

// ---- parts ----------------------------------------------------------------------------------------------------------------

// A long recording in parts, all at once: a part turns the state S before it into Z + F S, Z what it makes of zeros and F what it
// makes of the columns of 1 (dim more columns). Those are put together here, part after part, and then every part runs from the
// state that it begins with; back it is Y + F^T R. That is 2.6 times the work on as many times the SMs as there are parts.
//
// A block goes through the parts with 16 columns: the state as terms in shared memory, a warp makes 16 of its values a part; F is read one
// part ahead. s.start: BACK: R behind each part but the last, else S before each part but the first.
template <int DP, bool BACK>
__global__ void __launch_bounds__(2 * DP) k_delta_join(const __grid_constant__ Delta s) {
    constexpr int kStride = DP + 8, kPlane = 16 * kStride, NS = 3;
    __shared__ __align__(16) bf16 sm[2][NS * kPlane];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3, d0 = 16 * warp;
    const int tiles_e = (s.E + 15) / 16, tile = blockIdx.x % tiles_e, rows = 16 * tiles_e * DP;
    const long long bh = blockIdx.x / tiles_e;
    const float* before = BACK ? s.glast : s.first;
    float x[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 16 * tile + g + 8 * (i >> 1), d = d0 + 8 * j + 2 * t4 + (i & 1);
            x[j][i] = before && d < s.D && e < s.E ? before[(bh * s.D + d) * s.E + e] : 0.f;
        }
    float f[DP / 16][2][4];                                  // right operands (k, n) of F or its transpose, n this warp's values
    const int written = (s.D + 15) / 16 * 16;                // rows of F that a part has
    const auto fetch = [&](int p) {
        const float* turn = s.turn + (bh * s.parts + p) * DP * DP;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kk = 16 * k + 2 * t4 + (i & 1) + 8 * (i >> 1), n = d0 + 8 * j + g;
                    f[k][j][i] = (BACK ? n : kk) < written ? turn[BACK ? n * DP + kk : kk * DP + n] : 0.f;
                }
    };
    fetch(BACK ? s.parts - 1 : 0);
    for (int i = 0; i + 1 < s.parts; ++i) {
        const int p = BACK ? s.parts - 1 - i : i;            // the part that is gone through
        bf16* now = sm[i & 1];
        uint32_t a[NS][4];
        left<NS>(x[0], x[1], a);
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint32_t*>(now + n * kPlane + (g + 8 * (e & 1)) * kStride + d0 + 2 * t4 + 8 * (e >> 1)) = a[n][e];
        uint32_t b[DP / 16][2][2][NS];
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) terms<NS>(f[k][j][2 * e], f[k][j][2 * e + 1], b[k][j][e]);
        if (i + 2 < s.parts) fetch(BACK ? p - 1 : p + 1);
        const float* own = s.own + (bh * s.parts + p) * rows + 16 * tile * DP;
        float z[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[j][e] = own[(g + 8 * (e >> 1)) * DP + d0 + 8 * j + 2 * t4 + (e & 1)];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) clear(x[j]);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
            for (int n = 0; n < NS; ++n) ldsm(a[n], smem_at(now + n * kPlane + 16 * k) + at_rows_m(lane, kStride));
#pragma unroll
            for (int m = 0; m < NS; ++m)
#pragma unroll
                for (int n = 0; n + m < NS; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) mma(x[j], a[n], b[k][j][0][m], b[k][j][1][m]);
        }
        float* to = s.start + (bh * s.parts + (BACK ? p - 1 : p + 1)) * rows + 16 * tile * DP;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[j][e] += z[j][e];
                to[(g + 8 * (e >> 1)) * DP + d0 + 8 * j + 2 * t4 + (e & 1)] = x[j][e];
            }
    }
}

}  // namespace
