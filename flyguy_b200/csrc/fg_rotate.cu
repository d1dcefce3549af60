// Position rotation of queries and keys, alone or with the norms of each head in the same pass, and the gradients.
//
//   r = 1 / sqrt(mean(x^2) + eps), z = x r w, y = pairs of z turned: (a, b) -> A (a cos - b sin, b cos + a sin)
//   g = gy turned back (same A): gw = sum over rows of g x r,  gx = r (g w - x r mean(g w x r))
//
// A tick's angle is position * turns[i] / 2^64 of a turn: the 64-bit product wraps, which drops whole turns exactly, so
// the angle is as good at position 2^40 as at 0 (an fp32 product of position and frequency is off by 0.06 rad at 10^6).
// Its upper 32 bits give the nearest quarter turn and what is left, at most pi / 4 either way, for which the Taylor series
// of sine and cosine up to x^9 and x^8 are good to 2.5e-8.
#include "fg_memory.cuh"

namespace {
using namespace fgm;

constexpr int kWarps = 8;

struct Side {
    const char* x;
    char* y;
    const char* gy;
    char* gx;
    long long xs[3], ys[3], gys[3], gxs[3];   // strides of batch, tick, head, in values
    const float* w;
    float* gw;
    long long w_head;
    int heads;
};
struct Rotate {
    Side s[2];
    const long long* turns;
    const void* positions;
    long long pos_batch, pos_tick;
    int pos8, interleaved, norm;
    long long batch, ticks;
    int dim, turned;
    float eps, amplitude;
};

__device__ __forceinline__ long long position(const Rotate& a, long long b, long long t) {
    if (!a.positions) return t;
    const long long i = b * a.pos_batch + t * a.pos_tick;
    return a.pos8 ? static_cast<const long long*>(a.positions)[i] : static_cast<const int*>(a.positions)[i];
}
// cosine and sine of u / 2^32 of a turn, times `amplitude`
__device__ __forceinline__ void turned(uint32_t u, float amplitude, float& c, float& s) {
    const uint32_t quarter = (u + 0x20000000u) >> 30;
    const float x = (float)(int)(u - (quarter << 30)) * 1.46291807926715968e-9f, y = x * x;   // 2 pi / 2^32
    float sine = fmaf(y, 1.f / 362880, -1.f / 5040);
    sine = fmaf(y, sine, 1.f / 120);
    sine = fmaf(y, sine, -1.f / 6);
    sine = fmaf(y * x, sine, x);
    float cosine = fmaf(y, 1.f / 40320, -1.f / 720);
    cosine = fmaf(y, cosine, 1.f / 24);
    cosine = fmaf(y, cosine, -0.5f);
    cosine = fmaf(y, cosine, 1.f);
    const float p = quarter & 1 ? sine : cosine, q = quarter & 1 ? cosine : sine;
    c = (quarter + 1) & 2 ? -amplitude * p : amplitude * p;
    s = quarter & 2 ? -amplitude * q : amplitude * q;
}
__device__ __forceinline__ uint32_t upper(long long pos, unsigned long long turns) {
    return (uint32_t)(((unsigned long long)pos * turns) >> 32);
}
__device__ __forceinline__ void angle(const Rotate& a, long long pos, int i, float& c, float& s) {
    turned(upper(pos, (unsigned long long)__ldg(&a.turns[i])), a.amplitude, c, s);
}
__device__ __forceinline__ void pair_of(const Rotate& a, int i, int& p, int& q) {
    p = a.interleaved ? 2 * i : i;
    q = a.interleaved ? 2 * i + 1 : i + a.turned / 2;
}

struct Row {
    const Side* s;
    long long b, t;
    int h;
};
// row number -> queries first, then keys; a row is one head of one tick
__device__ __forceinline__ Row row_of(const Rotate& a, long long row) {
    Row r;
    const long long nq = a.batch * a.ticks * a.s[0].heads;
    r.s = &a.s[row >= nq];
    if (row >= nq) row -= nq;
    const long long tick = row / r.s->heads;
    r.h = (int)(row - tick * r.s->heads);
    r.b = tick / a.ticks;
    r.t = tick - r.b * a.ticks;
    return r;
}
template <class T>
__device__ __forceinline__ T* at(const char* p, const long long (&st)[3], const Row& r) {
    return reinterpret_cast<T*>(const_cast<char*>(p)) + r.b * st[0] + r.t * st[1] + r.h * st[2];
}

// Any size, stride and alignment: a warp per row, a lane per pair, the row read twice (the second time from L1). Bound by its
// narrow loads and by the angles, formed anew for each head: 32 recordings of 2,048 ticks, 8 + 8 heads of 128 in fp16 take
// 656 us, in whole units (below) 121.
template <class T>
__global__ void __launch_bounds__(32 * kWarps) k_rotate_any(const __grid_constant__ Rotate a, long long rows) {
    const int lane = threadIdx.x & 31;
    for (long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); row < rows;
         row += (long long)gridDim.x * kWarps) {
        const Row r = row_of(a, row);
        const T* x = at<const T>(r.s->x, r.s->xs, r);
        T* y = at<T>(r.s->y, r.s->ys, r);
        const float* w = r.s->w ? r.s->w + r.h * r.s->w_head : nullptr;
        float n = 1.f;
        if (a.norm) {
            float s = 0.f;
            for (int i = lane; i < a.dim; i += 32) s = fmaf(to_f(x[i]), to_f(x[i]), s);
            n = 1.f / sqrtf(warp_sum(s) / (float)a.dim + a.eps);
        }
        const long long pos = position(a, r.b, r.t);
        for (int i = lane; i < a.turned / 2; i += 32) {
            int p, q;
            float c, s;
            pair_of(a, i, p, q);
            angle(a, pos, i, c, s);
            const float u = to_f(x[p]) * n * (w ? w[p] : 1.f), v = to_f(x[q]) * n * (w ? w[q] : 1.f);
            y[p] = from_f<T>(u * c - v * s);
            y[q] = from_f<T>(v * c + u * s);
        }
        for (int i = a.turned + lane; i < a.dim; i += 32) y[i] = from_f<T>(to_f(x[i]) * n * (w ? w[i] : 1.f));
    }
}

// gradient of a row's value i before the rotation
template <class T>
__device__ __forceinline__ float turned_back(const Rotate& a, const T* gy, long long pos, int i) {
    if (i >= a.turned) return to_f(gy[i]);
    const int half = a.turned / 2;
    const int pair = a.interleaved ? i >> 1 : (i < half ? i : i - half);
    int p, q;
    float c, s;
    pair_of(a, pair, p, q);
    angle(a, pos, pair, c, s);
    return i == p ? to_f(gy[p]) * c + to_f(gy[q]) * s : to_f(gy[q]) * c - to_f(gy[p]) * s;
}

// gx; with the norm each row's n = 1 / sqrt(..) is kept for k_rotate_gw_any
template <class T>
__global__ void __launch_bounds__(32 * kWarps) k_rotate_bwd_any(const __grid_constant__ Rotate a, long long rows,
                                                                float* __restrict__ norms) {
    const int lane = threadIdx.x & 31;
    for (long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); row < rows;
         row += (long long)gridDim.x * kWarps) {
        const Row r = row_of(a, row);
        const T* gy = at<const T>(r.s->gy, r.s->gys, r);
        T* gx = at<T>(r.s->gx, r.s->gxs, r);
        const long long pos = position(a, r.b, r.t);
        if (!a.norm) {
            for (int i = lane; i < a.dim; i += 32) gx[i] = from_f<T>(turned_back(a, gy, pos, i));
            continue;
        }
        const T* x = at<const T>(r.s->x, r.s->xs, r);
        const float* w = r.s->w ? r.s->w + r.h * r.s->w_head : nullptr;
        float s = 0.f, m = 0.f;
        for (int i = lane; i < a.dim; i += 32) {
            const float v = to_f(x[i]);
            s = fmaf(v, v, s);
            m = fmaf(turned_back(a, gy, pos, i) * (w ? w[i] : 1.f), v, m);
        }
        const float n = 1.f / sqrtf(warp_sum(s) / (float)a.dim + a.eps);
        m = warp_sum(m) * n / (float)a.dim;
        for (int i = lane; i < a.dim; i += 32)
            gx[i] = from_f<T>(n * (turned_back(a, gy, pos, i) * (w ? w[i] : 1.f) - to_f(x[i]) * n * m));
        if (norms && lane == 0) norms[row] = n;
    }
}

// part[split][set][i] = sum over the split's ticks (and, with one set of weights for all heads, over the heads) of g x n
template <class T>
__global__ void __launch_bounds__(128) k_rotate_gw_any(const __grid_constant__ Rotate a, int side,
                                                       const float* __restrict__ norms, float* __restrict__ part,
                                                       int sets, int splits) {
    const int i = blockIdx.x * 128 + threadIdx.x, set = blockIdx.y, split = blockIdx.z;
    if (i >= a.dim) return;
    const Side& s = a.s[side];
    const long long ticks = a.batch * a.ticks, per = (ticks + splits - 1) / splits;
    const long long row0 = side ? ticks * a.s[0].heads : 0;
    float sum = 0.f;
    for (long long tick = split * per; tick < min(ticks, (split + 1) * per); ++tick) {
        Row r;
        r.s = &s;
        r.b = tick / a.ticks;
        r.t = tick - r.b * a.ticks;
        const long long pos = position(a, r.b, r.t);
        for (int h = sets > 1 ? set : 0; h < (sets > 1 ? set + 1 : s.heads); ++h) {
            r.h = h;
            sum = fmaf(turned_back(a, at<const T>(s.gy, s.gys, r), pos, i) * to_f(at<const T>(s.x, s.xs, r)[i]),
                       norms[row0 + tick * s.heads + h], sum);
        }
    }
    part[((long long)split * sets + set) * a.dim + i] = sum;
}
// gw = the splits' sums added in a fixed order: 32 warps each take every 32nd split of 32 values, then their sums in turn
struct SumSide {
    const float* part;
    float* gw;
    int n, splits;
};
__global__ void __launch_bounds__(1024) k_rotate_gw_sum(const SumSide queries, const SumSide keys) {
    __shared__ float sums[32][33];
    const SumSide a = blockIdx.y ? keys : queries;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (i < a.n) {
#pragma unroll 4
        for (int k = w; k < a.splits; k += 32) s += a.part[(long long)k * a.n + i];
    }
    sums[w][lane] = s;
    __syncthreads();
    if (w || i >= a.n) return;
#pragma unroll
    for (int k = 1; k < 32; ++k) s += sums[k][lane];
    a.gw[i] = s;
}

// ---- rows of whole 16-byte units ------------------------------------------------------------------------------------
//
// A block takes a few ticks of the queries, or of the keys, at a time. Its 256 threads form the ticks' angles once into
// shared memory; then every group of 2^k lanes takes heads of one tick, each lane two 16-byte units of a head: partners of
// the "half" layout, or any two. A lane's pairs are its own, so the rotation needs no exchange, the norm a few shuffles, and
// every value is read and written once. The lane's angles and weights stay in registers over its heads: fetched for each
// head they are three times the bytes of the values.
//
// The bound is the memory: 2 passes over the values forward (read, write), 3 back. What it takes to get near it: kAhead
// heads of each lane are on their way into shared memory at any time (a lane reads only what it asked for itself, so no
// barrier is needed), and the arithmetic is done on pairs of floats, for the kernel is half bound by its instructions. In
// bf16, half layout, 128 recordings of 128 ticks, 16 + 4 heads of 128, forward and back with the sums of gw: 42 and 75 us,
// where one head ahead in registers takes 49 and 99, and a row for each group, with its angles and weights fetched anew,
// 73 and 95; the bytes alone are 26 and 39 us. In fp16, 32 recordings of 2,048 ticks, 8 + 8 heads of 128, the first 96
// values turned as neighbours: 118 us (bytes: 82); where the lane's two units are neighbours too, 182.

// 16 bytes of T as pairs of floats, n values in all
template <class T>
struct Unit {
    static constexpr int n = 16 / sizeof(T), pairs = n / 2;
};
__device__ __forceinline__ uint64_t pair_of_bits(uint32_t v, __nv_bfloat16) {
    return two(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint64_t pair_of_bits(uint32_t v, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return two(f.x, f.y);
}
__device__ __forceinline__ uint32_t bits_of_pair(uint64_t x, __nv_bfloat16) {
    float a, b;
    halves(x, a, b);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t bits_of_pair(uint64_t x, __half) {
    float a, b;
    halves(x, a, b);
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <class T>
__device__ __forceinline__ void from_unit(const uint4& u, uint64_t (&v)[Unit<T>::pairs]) {
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
        v[0] = two(__uint_as_float(r[0]), __uint_as_float(r[1]));
        v[1] = two(__uint_as_float(r[2]), __uint_as_float(r[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pair_of_bits(r[i], T());
    }
}
template <class T>
__device__ __forceinline__ void store_unit(T* p, const uint64_t (&v)[Unit<T>::pairs]) {
    uint32_t r[4];
    if constexpr (sizeof(T) == 4) {
        float a, b, c, d;
        halves(v[0], a, b);
        halves(v[1], c, d);
        r[0] = __float_as_uint(a); r[1] = __float_as_uint(b); r[2] = __float_as_uint(c); r[3] = __float_as_uint(d);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = bits_of_pair(v[i], T());
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
}
// values of p and of q turned by the angles c, s (with `minus` = -s), value i of p with value i of q
template <int P>
__device__ __forceinline__ void turn_apart(uint64_t (&p)[P], uint64_t (&q)[P], const uint64_t (&c)[P], const uint64_t (&s)[P],
                                           const uint64_t (&minus)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const uint64_t u = p[i], v = q[i];
        p[i] = fma2(u, c[i], mul2(v, minus[i]));
        q[i] = fma2(v, c[i], mul2(u, s[i]));
    }
}
// neighbours of one unit, by its half of the angles
template <int HALF, int P>
__device__ __forceinline__ void turn_neighbours(uint64_t (&p)[P], const uint64_t (&c)[P], const uint64_t (&s)[P]) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
        float c0, c1, s0, s1, a, b;
        halves(c[HALF * P / 2 + i], c0, c1);
        halves(s[HALF * P / 2 + i], s0, s1);
        halves(p[2 * i], a, b);
        p[2 * i] = two(a * c0 - b * s0, b * c0 + a * s0);
        halves(p[2 * i + 1], a, b);
        p[2 * i + 1] = two(a * c1 - b * s1, b * c1 + a * s1);
    }
}

enum { kForward, kBackward, kBackwardW, kBackwardEach };     // the last two with gw: one set of weights, one for each head

struct UnitPlan {
    int per[2], blocks[2];                                   // ticks at a time (powers of 2) and blocks, for queries and keys
    int lanes;                                               // of a group
    uint32_t by_ticks;                                       // 2^32 / ticks, rounded up
};
constexpr int kAhead = 4;                                    // heads whose values are on their way into shared memory
template <bool NORM, int MODE>
constexpr int kUnits = MODE != kForward && NORM ? 4 : 2;     // 16-byte units that a lane reads of a head
// 16 bytes, or zeros: nothing is read then
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
// n / d with r = 2^32 / d rounded up, n < 2^30: at most one too many
__device__ __forceinline__ int divided(int n, int d, uint32_t r) {
    if (d == 1) return n;
    const int q = (int)__umulhi((uint32_t)n, r);
    return q * d > n ? q - 1 : q;
}

template <class T, bool INTER, bool NORM, int MODE>
__global__ void __launch_bounds__(256, MODE != kForward && NORM ? 2 : 3) k_rotate_units(const __grid_constant__ Rotate a,
                                                                                 const UnitPlan plan,
                                                                                 float* __restrict__ part) {
    constexpr int N = Unit<T>::n, P = Unit<T>::pairs, U = kUnits<NORM, MODE>;
    extern __shared__ __align__(16) float all_shared[];      // [kAhead][U][256] units, then what follows
    float* shared = all_shared + kAhead * U * 256 * 4;
    const int side = (int)blockIdx.x >= plan.blocks[0], block = side ? (int)blockIdx.x - plan.blocks[0] : (int)blockIdx.x;
    const Side s = side ? a.s[1] : a.s[0];                   // (by selection: an index into the arguments is a load each time)
    const int heads = s.heads, per = side ? plan.per[1] : plan.per[0], half_turn = a.turned / 2;
    float2* angles = reinterpret_cast<float2*>(shared);      // [2][per][turned / 2]
    float* sums = shared + 4 * per * half_turn;              // kBackwardEach: [heads][dim]
    const int tid = threadIdx.x, lane = tid & (plan.lanes - 1), group = tid / plan.lanes, groups = 256 / plan.lanes;
    const bool busy = lane < a.dim / (2 * N);
    // the lane's two units of a head: partners, or, where pairs are neighbours or not turned at all, any two. Lanes side by
    // side take units side by side: 32-byte sectors that two loads or stores take a half of each cost twice.
    const bool partners = !INTER && busy && lane * N < half_turn;
    const int rest = lane - half_turn / N, left = (a.dim - a.turned) / 2;
    const int u0 = INTER || partners ? lane * N : a.turned + rest * N;
    const int u1 = INTER ? u0 + a.dim / 2 : partners ? u0 + half_turn : u0 + left;
    const bool turns0 = INTER ? busy && u0 < a.turned : partners, turns1 = INTER ? busy && u1 < a.turned : partners;
    // groups of one tick share its heads; with sums for each head there is one tick, so that a head stays with its group
    const int share = groups / per, j = group / share, first = group - j * share;
    const int total = (int)(a.batch * a.ticks), ticks = (int)a.ticks;
    const float inverse = 1.f / (float)a.dim;
    uint64_t w0[P], w1[P], gw0[P], gw1[P];
#pragma unroll
    for (int k = 0; k < P; ++k) w0[k] = w1[k] = two(1.f, 1.f), gw0[k] = gw1[k] = 0;
    auto weights = [&](int h) {
        const float4* w = reinterpret_cast<const float4*>(s.w + h * s.w_head);
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const float4 f = __ldg(w + u0 / 4 + k), g = __ldg(w + u1 / 4 + k);
            w0[2 * k] = two(f.x, f.y); w0[2 * k + 1] = two(f.z, f.w);
            w1[2 * k] = two(g.x, g.y); w1[2 * k + 1] = two(g.z, g.w);
        }
    };
    if (NORM && s.w && !s.w_head && busy) weights(0);
    if (MODE == kBackwardEach) {
        for (int i = tid; i < heads * a.dim; i += 256) sums[i] = 0.f;
        __syncthreads();
    }
    // the thread's first angle of the block's ticks, and how far on its next is
    const int my_tick = half_turn ? tid / half_turn : 0, my_pair = tid - my_tick * half_turn;
    const int more_ticks = half_turn ? 256 / half_turn : 0, more_pairs = 256 - more_ticks * half_turn;
    const long long x_head = s.xs[2], gy_head = s.gys[2], to_head = MODE == kForward ? s.ys[2] : s.gxs[2];
    constexpr uint32_t kSlot = U * 256 * 16;
    const T *x_base = reinterpret_cast<const T*>(s.x), *gy_base = reinterpret_cast<const T*>(s.gy);
    const uint32_t my_slot = (uint32_t)__cvta_generic_to_shared(all_shared) + tid * 16;
    const int step = (side ? plan.blocks[1] : plan.blocks[0]) * per;
    for (int tick0 = block * per, turn_no = 0; tick0 < total; tick0 += step, ++turn_no) {
        const int n = min(per, total - tick0);
        const bool there = busy && j < n;
        const int mine = tick0 + (there ? j : 0), b = divided(mine, ticks, plan.by_ticks), t = mine - b * ticks;
        const T* x_at = reinterpret_cast<const T*>(s.x) + b * s.xs[0] + t * s.xs[1] + first * x_head;
        const T* gy_at = reinterpret_cast<const T*>(s.gy) + b * s.gys[0] + t * s.gys[1] + first * gy_head;
        T* to = MODE == kForward ? reinterpret_cast<T*>(s.y) + b * s.ys[0] + t * s.ys[1] + first * to_head
                                 : reinterpret_cast<T*>(s.gx) + b * s.gxs[0] + t * s.gxs[1] + first * to_head;
        const int mine_heads = there ? heads : 0;
        int ask = first;                                      // the head that is asked for next, and its place
        uint32_t ask_slot = my_slot;
        auto fetch = [&]() {                                  // (zeros where there is none)
            const bool some = ask < mine_heads;
            if (MODE == kForward || NORM) {
                copy16(ask_slot, some ? x_at + u0 : x_base, some);
                copy16(ask_slot + 256 * 16, some ? x_at + u1 : x_base, some);
            }
            if (MODE != kForward) {
                copy16(ask_slot + (U - 2) * 256 * 16, some ? gy_at + u0 : gy_base, some);
                copy16(ask_slot + (U - 1) * 256 * 16, some ? gy_at + u1 : gy_base, some);
            }
            copies_end();
            x_at += share * x_head;
            gy_at += share * gy_head;
            ask += share;
            ask_slot = ask_slot == my_slot + (kAhead - 1) * kSlot ? my_slot : ask_slot + kSlot;
        };
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) fetch();         // (on their way while the angles are formed)
        float2* here_angles = angles + (turn_no & 1) * per * half_turn;
        for (int i = tid, at = my_tick, pair = my_pair; i < n * half_turn; i += 256) {
            const int tick = tick0 + at, tb = divided(tick, ticks, plan.by_ticks);
            float2 cs;
            angle(a, position(a, tb, tick - tb * ticks), pair, cs.x, cs.y);
            here_angles[i] = cs;
            at += more_ticks;
            pair += more_pairs;
            if (pair >= half_turn) pair -= half_turn, ++at;
        }
        __syncthreads();                                      // (two sets of angles: nobody is a whole turn ahead)
        uint64_t c[P], sn[P], minus[P];                       // the lane's N angles (back: turned the other way)
#pragma unroll
        for (int k = 0; k < P; ++k) c[k] = sn[k] = minus[k] = 0;   // (a group without a tick adds zeros to gw)
        if (turns0 && there) {                                // (partners have one set, of N pairs; neighbours two of N / 2)
            const float4* of0 = reinterpret_cast<const float4*>(here_angles + j * half_turn + (INTER ? u0 / 2 : u0));
            const float4* of1 = reinterpret_cast<const float4*>(here_angles + j * half_turn + u1 / 2) - P / 2;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                if (INTER && k >= P / 2 && !turns1) break;
                const float4 f = INTER && k >= P / 2 ? of1[k] : of0[k];
                c[k] = two(f.x, f.z);
                sn[k] = MODE == kForward ? two(f.y, f.w) : two(-f.y, -f.w);
                minus[k] = MODE == kForward ? two(-f.y, -f.w) : two(f.y, f.w);
            }
        }
        auto turn = [&](uint64_t (&p)[P], uint64_t (&q)[P]) {
            if (INTER) {
                if (turns0) turn_neighbours<0, P>(p, c, sn);
                if (turns1) turn_neighbours<1, P>(q, c, sn);
            } else if (partners) {
                turn_apart<P>(p, q, c, sn, minus);
            }
        };
        int slot = 0;
        for (int h = first; h < (heads + share - 1) / share * share; h += share) {
            fetch();                                          // (into the slot of the head before, which is used up)
            copies_wait<kAhead - 1>();
            const uint4* got = reinterpret_cast<const uint4*>(all_shared) + tid + slot;
            slot = slot == (kAhead - 1) * U * 256 ? 0 : slot + U * 256;
            const bool here = h < mine_heads;
            uint64_t p[P], q[P], x[P], y[P];
            if (MODE == kForward || NORM) {
                from_unit<T>(got[0], x);
                from_unit<T>(got[256], y);
            }
            if (MODE != kForward) {
                from_unit<T>(got[(U - 2) * 256], p);
                from_unit<T>(got[(U - 1) * 256], q);
                turn(p, q);
            }
            if (NORM && s.w && s.w_head && here) weights(h);
            if (NORM) {
                uint64_t sq2 = 0, m2 = 0;
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    sq2 = fma2(x[k], x[k], fma2(y[k], y[k], sq2));
                    if (MODE != kForward) {
                        m2 = fma2(mul2(p[k], w0[k]), x[k], fma2(mul2(q[k], w1[k]), y[k], m2));
                    }
                }
                float sq = sum2(sq2), m = MODE != kForward ? sum2(m2) : 0.f;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    if (o >= plan.lanes) break;
                    sq += __shfl_xor_sync(0xffffffffu, sq, o);
                    if (MODE != kForward) m += __shfl_xor_sync(0xffffffffu, m, o);
                }
                const float norm = rsqrtf(fmaf(sq, inverse, a.eps));
                const uint64_t norm2 = two(norm, norm);
                if (MODE == kForward) {
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        x[k] = mul2(x[k], mul2(norm2, w0[k]));
                        y[k] = mul2(y[k], mul2(norm2, w1[k]));
                    }
                } else {
                    // gx = norm (g w - x norm^2 mean(g w x))
                    const float mean = -m * norm * norm * inverse;
                    const uint64_t mean2 = two(mean, mean);
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        if (MODE == kBackwardW) {
                            gw0[k] = fma2(p[k], mul2(x[k], norm2), gw0[k]);
                            gw1[k] = fma2(q[k], mul2(y[k], norm2), gw1[k]);
                        }
                        if (MODE == kBackwardEach && here) {
                            float2* at0 = reinterpret_cast<float2*>(sums + h * a.dim + u0 + 2 * k);
                            float2* at1 = reinterpret_cast<float2*>(sums + h * a.dim + u1 + 2 * k);
                            float f, g;
                            halves(fma2(p[k], mul2(x[k], norm2), two(at0->x, at0->y)), f, g);
                            *at0 = make_float2(f, g);
                            halves(fma2(q[k], mul2(y[k], norm2), two(at1->x, at1->y)), f, g);
                            *at1 = make_float2(f, g);
                        }
                        p[k] = mul2(norm2, fma2(x[k], mean2, mul2(p[k], w0[k])));
                        q[k] = mul2(norm2, fma2(y[k], mean2, mul2(q[k], w1[k])));
                    }
                }
            }
            if (!here) continue;
            if (MODE == kForward) {
                turn(x, y);
                store_unit(to + u0, x);
                store_unit(to + u1, y);
            } else {
                store_unit(to + u0, p);
                store_unit(to + u1, q);
            }
            to += share * to_head;
        }
        // what was asked for past the last head (zeros) lands before the next ticks' copies go to the same places: copies are
        // in no order among themselves
        copies_wait<0>();
    }
    if (MODE == kBackwardW) {
        // the groups' sums in turn: part [block][dim], the queries' blocks first
        float* all = shared;                                  // [groups][dim]
        __syncthreads();
        if (busy) {
#pragma unroll
            for (int k = 0; k < P; ++k) {
                float f, g;
                halves(gw0[k], f, g);
                *reinterpret_cast<float2*>(all + group * a.dim + u0 + 2 * k) = make_float2(f, g);
                halves(gw1[k], f, g);
                *reinterpret_cast<float2*>(all + group * a.dim + u1 + 2 * k) = make_float2(f, g);
            }
        }
        __syncthreads();
        for (int i = tid; i < a.dim; i += 256) {
            float sum = 0.f;
            for (int g = 0; g < groups; ++g) sum += all[g * a.dim + i];
            part[(long long)blockIdx.x * a.dim + i] = sum;
        }
    }
    if (MODE == kBackwardEach) {                              // part [block][heads][dim], the queries' blocks first
        __syncthreads();
        float* to = part + ((long long)block * heads + (side ? (long long)plan.blocks[0] * a.s[0].heads : 0)) * a.dim;
        for (int i = tid; i < heads * a.dim; i += 256) to[i] = sums[i];
    }
}

constexpr int kSplits = kSms * 4;                            // blocks with sums of their own, at most

void strides(long long (&to)[3], const fg_ticks& t) {
    to[0] = t.batch;
    to[1] = t.tick;
    to[2] = t.head;
}

Rotate checked(const fg_rotate_args* g, bool backward) {
    need(g, "fg_norm_rotate: no arguments");
    need(g->batch >= 0 && g->ticks >= 0 && g->heads[0] >= 0 && g->heads[1] >= 0, "fg_norm_rotate: a negative size");
    need(g->dim > 0 && g->dim <= 65536, "fg_norm_rotate: dim must be 1 to 65536");
    need(g->turned >= 0 && g->turned % 2 == 0 && g->turned <= g->dim,
         "fg_norm_rotate: turned must be even and at most dim");
    need(!g->turned || g->turns, "fg_norm_rotate: turned values need turns");
    need(!g->positions || g->pos_bytes == 4 || g->pos_bytes == 8, "fg_norm_rotate: positions are of 4 or 8 bytes");
    need(!g->norm || (float)g->eps > 0, "fg_norm_rotate: eps must be positive");
    need(g->type >= FG_F32 && g->type <= FG_F16, "fg_norm_rotate: unknown type");
    Rotate a{};
    for (int i = 0; i < 2; ++i) {
        Side& s = a.s[i];
        const bool used = g->heads[i] && g->batch && g->ticks;
        need(g->heads[i] < (1 << 24), "fg_norm_rotate: too many heads");
        s.x = static_cast<const char*>(g->x[i].p);
        s.y = static_cast<char*>(g->y[i].p);
        s.gy = static_cast<const char*>(g->gy[i].p);
        s.gx = static_cast<char*>(g->gx[i].p);
        need(!used || (backward ? s.gy && s.gx && (s.x || !g->norm) : s.x && s.y), "fg_norm_rotate: null pointer");
        strides(s.xs, g->x[i]);
        strides(s.ys, g->y[i]);
        strides(s.gys, g->gy[i]);
        strides(s.gxs, g->gx[i]);
        s.w = g->norm ? g->w[i] : nullptr;
        s.gw = g->norm ? g->gw[i] : nullptr;
        s.w_head = g->w_head[i];
        need(s.w_head == 0 || s.w_head >= g->dim, "fg_norm_rotate: heads' weights overlap");
        s.heads = (int)g->heads[i];
    }
    a.turns = g->turns;
    a.positions = g->positions;
    a.pos_batch = g->pos_batch;
    a.pos_tick = g->pos_tick;
    a.pos8 = g->pos_bytes == 8;
    a.interleaved = g->interleaved != 0;
    a.norm = g->norm != 0;
    a.batch = g->batch;
    a.ticks = g->ticks;
    a.dim = (int)g->dim;
    a.turned = (int)g->turned;
    a.eps = (float)g->eps;
    a.amplitude = (float)g->amplitude;
    return a;
}

long long rows_of(const fg_rotate_args* g) { return g->batch * g->ticks * (g->heads[0] + g->heads[1]); }
long long sets_of(const fg_rotate_args* g, int i) { return g->w_head[i] ? g->heads[i] : 1; }

// Whether heads have weights of their own, and whether k_rotate_units forms their sums: those of one set of weights for some
// heads and sets of their own for others go the general way.
bool each_head(const fg_rotate_args* g) { return g->w_head[0] || g->w_head[1]; }
bool sums_of_each(const fg_rotate_args* g) {
    for (int i = 0; i < 2; ++i)
        if (g->gw[i] && g->heads[i] && !g->w_head[i]) return false;
    return each_head(g) && (g->heads[0] + g->heads[1]) * g->dim * 4 <= 64 * 1024;
}

// The rows' norms, then every block's sums. In sums_of_each calls a block leaves sums for each head of its side, also of a
// side whose weights are shared, frozen or absent.
long long work_bytes(const fg_rotate_args* g) {
    if (!g->norm || (!g->gw[0] && !g->gw[1])) return 0;
    const bool all = sums_of_each(g);
    long long sets = 1;
    for (int i = 0; i < 2; ++i)
        if (all || (g->gw[i] && g->w_head[i])) sets = std::max(sets, g->heads[i]);
    const long long blocks = std::min<long long>(kSplits, 2 * g->batch * g->ticks) + 2;
    return (rows_of(g) + 3) / 4 * 16 + sets * g->dim * blocks * 4;
}

unsigned blocks_for(long long rows) {
    return (unsigned)std::max<long long>(1, std::min<long long>((rows + kWarps - 1) / kWarps, 1 << 20));
}

bool aligned(const void* p, const long long (&st)[3], long long unit) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] % unit == 0 && st[1] % unit == 0 && st[2] % unit == 0;
}
// whether rows are whole pairs of 16-byte units, each turned as a whole or not at all, partners in units of their own
bool has_units(const Rotate& a, int size, bool backward) {
    const int unit = 16 / size;
    if (a.dim % (2 * unit) || a.turned % (a.interleaved ? unit : 2 * unit) || a.dim / (2 * unit) > 32 || a.batch * a.ticks >= (1ll << 30)) return false;
    for (const Side& s : a.s) {
        if (!s.heads) continue;
        if ((!backward || a.norm) && !aligned(s.x, s.xs, unit)) return false;
        if (backward ? !aligned(s.gy, s.gys, unit) || !aligned(s.gx, s.gxs, unit) : !aligned(s.y, s.ys, unit)) return false;
        if (s.w && (reinterpret_cast<uintptr_t>(s.w) % 16 || s.w_head % 4)) return false;
    }
    return true;
}
template <class T, bool INTER, bool NORM, int MODE>
void launch_units(const Rotate& a, float* part, UnitPlan& plan, cudaStream_t st) {
    const int items = a.dim / (2 * Unit<T>::n), half = a.turned / 2, total = (int)(a.batch * a.ticks);
    const int rows = a.s[0].heads + a.s[1].heads;
    plan = UnitPlan{{1, 1}, {0, 0}, 1, (uint32_t)(((1ull << 32) + a.ticks - 1) / a.ticks)};
    while (plan.lanes < items) plan.lanes *= 2;
    const int groups = 256 / plan.lanes, most = MODE >= kBackwardW ? kSplits : kSms * 12;
    size_t bytes = 0;
    for (int i = 0; i < 2; ++i) {
        const int heads = a.s[i].heads;
        if (!heads) continue;
        // a group takes a tick's heads one after another, unless the ticks are too few to give each SM two blocks: what a
        // tick costs by itself (its place, its angles) is spread over its heads. With the sizes above 2 blocks an SM take
        // 42 and 75 us, 8 take 57 and 87; 2,048 angles twice are 32 KB of an SM's shared memory a block.
        int per = MODE == kBackwardEach ? 1 : groups;
        while (per > 1 && ((total + per - 1) / per < kSms * 2 || (size_t)per * half > 2048)) per /= 2;
        plan.per[i] = per;
        bytes = std::max(bytes, (size_t)per * half * 16 + (MODE == kBackwardEach ? (size_t)heads * a.dim * 4 : 0));
        plan.blocks[i] = std::max(1, std::min((total + per - 1) / per, (int)((long long)most * heads / rows)));
    }
    if (MODE == kBackwardW) bytes = std::max(bytes, (size_t)groups * a.dim * 4);
    bytes += kAhead * kUnits<NORM, MODE> * 256 * 16;
    auto* k = k_rotate_units<T, INTER, NORM, MODE>;
    // (the most any sizes ask for, once: set to each call's own, another thread's call could lower it before this one's launch)
    constexpr int most_bytes = 64 * 1024 + 2048 * 16 + kAhead * kUnits<NORM, MODE> * 256 * 16;
    need(bytes <= (size_t)most_bytes, "fg_norm_rotate: the tiles do not fit shared memory");
    static OnEachDevice here;
    here.first(current_device(), [] { allow_shared(k_rotate_units<T, INTER, NORM, MODE>, most_bytes); });
    k<<<plan.blocks[0] + plan.blocks[1], 256, bytes, st>>>(a, plan, part);
    MCK(cudaGetLastError());
}
template <class T, int MODE>
void launch_units(const Rotate& a, float* part, UnitPlan& plan, cudaStream_t st) {
    constexpr bool with_norm = MODE >= kBackwardW;            // (sums of gw are the norm's)
    if (a.norm) a.interleaved ? launch_units<T, true, true, MODE>(a, part, plan, st) : launch_units<T, false, true, MODE>(a, part, plan, st);
    else if constexpr (!with_norm) a.interleaved ? launch_units<T, true, false, MODE>(a, part, plan, st) : launch_units<T, false, false, MODE>(a, part, plan, st);
}

}  // namespace

extern "C" {

int fg_norm_rotate(const fg_rotate_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        const Rotate a = checked(g, false);
        const long long rows = rows_of(g);
        if (!rows) return 0;
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            cudaStream_t st = static_cast<cudaStream_t>(stream);
            UnitPlan plan;
            if (has_units(a, sizeof(T), false)) launch_units<T, kForward>(a, nullptr, plan, st);
            else k_rotate_any<T><<<blocks_for(rows), 32 * kWarps, 0, st>>>(a, rows);
        });
        MCK(cudaGetLastError());
        return 0;
    });
}

long long fg_norm_rotate_work(const fg_rotate_args* g) {
    return mem_guard([&]() -> long long {
        need(g, "fg_norm_rotate: no arguments");
        return work_bytes(g);
    });
}

int fg_norm_rotate_bwd(const fg_rotate_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        const Rotate a = checked(g, true);
        const long long rows = rows_of(g), need_bytes = work_bytes(g);
        need(!need_bytes || (g->work && g->work_bytes >= need_bytes), "fg_norm_rotate_bwd: the workspace is too small");
        need(reinterpret_cast<uintptr_t>(g->work) % 16 == 0, "fg_norm_rotate_bwd: the workspace is not 16-byte aligned");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        float* norms = need_bytes ? static_cast<float*>(g->work) : nullptr;
        for (int i = 0; i < 2; ++i)                           // (weights that no head has used)
            if (a.s[i].gw && !a.s[i].heads && !g->w_head[i]) MCK(cudaMemsetAsync(a.s[i].gw, 0, a.dim * sizeof(float), st));
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            float* part = norms ? norms + (rows + 3) / 4 * 4 : nullptr;
            const bool each = each_head(g), fits = !each || sums_of_each(g);
            if (rows && has_units(a, sizeof(T), true) && (!norms || fits)) {
                UnitPlan plan;
                if (!norms) launch_units<T, kBackward>(a, nullptr, plan, st);
                else if (each) launch_units<T, kBackwardEach>(a, part, plan, st);
                else launch_units<T, kBackwardW>(a, part, plan, st);
                if (norms) {
                    SumSide sums[2];
                    for (int i = 0; i < 2; ++i) {
                        const int n = (int)(each ? g->heads[i] : 1) * a.dim;
                        sums[i] = {i ? sums[0].part + (long long)plan.blocks[0] * sums[0].n : part, a.s[i].gw, n, plan.blocks[i]};
                    }
                    const int n0 = a.s[0].gw && a.s[0].heads ? sums[0].n : 0, n1 = a.s[1].gw && a.s[1].heads ? sums[1].n : 0;
                    sums[0].n = n0;
                    sums[1].n = n1;
                    if (n0 || n1) k_rotate_gw_sum<<<dim3((std::max(n0, n1) + 31) / 32, 2), 1024, 0, st>>>(sums[0], sums[1]);
                    MCK(cudaGetLastError());
                }
                return;
            }
            if (rows) k_rotate_bwd_any<T><<<blocks_for(rows), 32 * kWarps, 0, st>>>(a, rows, norms);
            MCK(cudaGetLastError());
            for (int i = 0; i < 2; ++i) {
                if (!a.s[i].gw || !a.s[i].heads) continue;
                const int sets = (int)sets_of(g, i), n = sets * a.dim;
                need(sets <= 65535, "fg_norm_rotate_bwd: too many heads with weights of their own");
                const int splits = (int)std::max<long long>(1, std::min<long long>(256, g->batch * g->ticks));
                const dim3 grid((a.dim + 127) / 128, sets, splits);
                k_rotate_gw_any<T><<<grid, 128, 0, st>>>(a, i, norms, part, sets, splits);
                k_rotate_gw_sum<<<dim3((n + 31) / 32, 1), 1024, 0, st>>>(SumSide{part, a.s[i].gw, n, splits}, SumSide{});
                MCK(cudaGetLastError());
            }
        });
        return 0;
    });
}

}  // extern "C"
