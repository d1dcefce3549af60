// Position rotation of queries and keys, alone or with the norms of each head in the same pass, and the gradients.
//
//   r = 1 / sqrt(mean(x^2) + eps), z = x r w, y = pairs of z turned: (a, b) -> A (a cos - b sin, b cos + a sin)
//   g = gy turned back (same A): gw = sum over rows of g x r,  gx = r (g w - x r mean(g w x r))
//
// A tick's angle is position * turns[i] / 2^64 of a turn: the 64-bit product wraps, which drops whole turns exactly, so
// the angle is as good at position 2^40 as at 0 (an fp32 product of position and frequency is off by 0.06 rad at 10^6).
// Its upper 32 bits, as a signed fraction of half a turn, go to sincospif.
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
__device__ __forceinline__ void angle(const Rotate& a, long long pos, int i, float& c, float& s) {
    const unsigned long long u = (unsigned long long)pos * (unsigned long long)__ldg(&a.turns[i]);
    sincospif((float)(int)(u >> 32) * 4.656612873077393e-10f, &s, &c);   // 2^-31: a full turn is 2
    c *= a.amplitude;
    s *= a.amplitude;
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

// Any size, stride and alignment: a warp per row, a lane per pair, the row read twice (the second time from L1).
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
// gw = the splits' sums added in a fixed order: 32 warps each take every 32nd split of 32 values, then their sums in turn.
// Values 0 .. n0 - 1 of a split go to gw0, those from `second` on to gw1.
__global__ void __launch_bounds__(1024) k_rotate_gw_sum(const float* __restrict__ part, float* __restrict__ gw0, int n0,
                                                        float* __restrict__ gw1, int second, int n1, int stride,
                                                        int splits) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    const bool one = gw0 && i < n0, two = gw1 && i >= second && i < second + n1;
    float s = 0.f;
    if (one || two) {
#pragma unroll 4
        for (int k = w; k < splits; k += 32) s += part[(long long)k * stride + i];
    }
    sums[w][lane] = s;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < 32; ++k) s += sums[k][lane];
    if (one) gw0[i] = s;
    if (two) gw1[i - second] = s;
}

// ---- rows of whole 16-byte units ------------------------------------------------------------------------------------
//
// A block takes a few ticks at a time: 256 threads form the ticks' angles once into shared memory (as many as one each),
// then every group of 2^k lanes takes some heads of one tick, each lane two 16-byte units of a head: the partners of the
// "half" layout (unit u and u + turned / 2), or two neighbours. A lane's pairs of values are its own, so the rotation needs
// no exchange, the norm a few shuffles, and every value is read and written once, 16 bytes a load. The lane's angles and
// weights stay in registers over its heads: fetched for each head they are three times the bytes of the values, and L1
// was the limit (128 recordings of 128 ticks, 16 + 4 heads of 128 in bf16: @@ us forward, @@ us back). The next head's
// values are asked for before the present one's are used.

template <class T>
struct Unit {                                                // 16 bytes of T as floats
    static constexpr int n = 16 / sizeof(T);
};
template <class T>
__device__ __forceinline__ void from_unit(const uint4& u, float (&v)[Unit<T>::n]) {
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
    } else {
        const T* t = reinterpret_cast<const T*>(r);
#pragma unroll
        for (int i = 0; i < Unit<T>::n; ++i) v[i] = to_f(t[i]);
    }
}
template <class T>
__device__ __forceinline__ void store_unit(T* p, const float (&v)[Unit<T>::n]) {
    uint32_t r[4];
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
    } else {
        T* t = reinterpret_cast<T*>(r);
#pragma unroll
        for (int i = 0; i < Unit<T>::n; ++i) t[i] = from_f<T>(v[i]);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
}
// (p[i], q[i]) turned by (c, s); INTER: the pairs are neighbours within p, then within q
template <bool INTER, int N>
__device__ __forceinline__ void turn(float (&p)[N], float (&q)[N], const float (&c)[N], const float (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float& a = INTER ? (i < N / 2 ? p[2 * i] : q[2 * i - N]) : p[i];
        float& b = INTER ? (i < N / 2 ? p[2 * i + 1] : q[2 * i + 1 - N]) : q[i];
        const float u = a, v = b;
        a = u * c[i] - v * s[i];
        b = v * c[i] + u * s[i];
    }
}

constexpr int kTicksMost = 8;

enum { kForward, kBackward, kBackwardW, kBackwardEach };     // the last two with gw: one set of weights, one for each head

struct UnitPlan {
    int per[2];                                              // ticks at a time, for queries and keys (powers of 2)
    int lanes;                                               // of a group
};

template <class T, bool INTER, bool NORM, int MODE>
__global__ void __launch_bounds__(256, MODE >= kBackwardW ? 2 : 3) k_rotate_units(const __grid_constant__ Rotate a,
                                                                                 const UnitPlan plan,
                                                                                 float* __restrict__ part) {
    constexpr int N = Unit<T>::n;
    extern __shared__ __align__(16) float shared[];
    const Side& s = a.s[blockIdx.y];
    const int heads = s.heads, per = plan.per[blockIdx.y], half_turn = a.turned / 2;
    float2* angles = reinterpret_cast<float2*>(shared);      // [2][per][turned / 2]
    float* sums = shared + 4 * per * half_turn;              // kBackwardEach: [heads][dim]
    const int tid = threadIdx.x, lane = tid & (plan.lanes - 1), group = tid / plan.lanes, groups = 256 / plan.lanes;
    const bool busy = lane < a.dim / (2 * N);
    // the lane's two units of a head, and its first pair
    const bool turns = busy && lane * N < half_turn;
    const int rest = lane - half_turn / N;
    const int u0 = !INTER && turns ? lane * N : !INTER ? a.turned + rest * 2 * N : lane * 2 * N;
    const int u1 = !INTER && turns ? u0 + half_turn : u0 + N;
    // groups of one tick share its heads; with sums for each head there is one tick, so that a head stays with its group
    const int share = groups / per, j = group / share, first = group - j * share;
    const int total = (int)(a.batch * a.ticks), ticks = (int)a.ticks;
    const float inverse = 1.f / (float)a.dim;
    float w0[N], w1[N], gw0[N], gw1[N];
#pragma unroll
    for (int k = 0; k < N; ++k) w0[k] = w1[k] = 1.f, gw0[k] = gw1[k] = 0.f;
    auto weights = [&](int h) {
        const float4* w = reinterpret_cast<const float4*>(s.w + h * s.w_head);
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const float4 f = __ldg(w + u0 / 4 + k), g = __ldg(w + u1 / 4 + k);
            w0[4 * k] = f.x; w0[4 * k + 1] = f.y; w0[4 * k + 2] = f.z; w0[4 * k + 3] = f.w;
            w1[4 * k] = g.x; w1[4 * k + 1] = g.y; w1[4 * k + 2] = g.z; w1[4 * k + 3] = g.w;
        }
    };
    if (NORM && s.w && !s.w_head && busy) weights(0);
    if (MODE == kBackwardEach) {
        for (int i = tid; i < heads * a.dim; i += 256) sums[i] = 0.f;
        __syncthreads();
    }
    for (int tick0 = blockIdx.x * per, turn_no = 0; tick0 < total; tick0 += gridDim.x * per, ++turn_no) {
        const int n = min(per, total - tick0);
        const bool there = busy && j < n;
        const int mine = tick0 + (there ? j : 0), b = mine / ticks, t = mine - b * ticks;
        const T* x_at = reinterpret_cast<const T*>(s.x) + b * s.xs[0] + t * s.xs[1];
        const T* gy_at = reinterpret_cast<const T*>(s.gy) + b * s.gys[0] + t * s.gys[1];
        T* to = MODE == kForward ? reinterpret_cast<T*>(s.y) + b * s.ys[0] + t * s.ys[1]
                                 : reinterpret_cast<T*>(s.gx) + b * s.gxs[0] + t * s.gxs[1];
        const long long to_head = MODE == kForward ? s.ys[2] : s.gxs[2];
        uint4 next[4];
        auto fetch = [&](int h) {
            if (!there || h >= heads) return;
            if (MODE == kForward || NORM) {
                next[0] = *reinterpret_cast<const uint4*>(x_at + h * s.xs[2] + u0);
                next[1] = *reinterpret_cast<const uint4*>(x_at + h * s.xs[2] + u1);
            }
            if (MODE != kForward) {
                next[2] = *reinterpret_cast<const uint4*>(gy_at + h * s.gys[2] + u0);
                next[3] = *reinterpret_cast<const uint4*>(gy_at + h * s.gys[2] + u1);
            }
        };
        fetch(first);                                         // (on its way while the angles are formed)
        float2* here_angles = angles + (turn_no & 1) * per * half_turn;
        for (int i = tid; i < n * half_turn; i += 256) {
            const int q = i / half_turn, pair = i - q * half_turn, tick = tick0 + q, tb = tick / ticks;
            float2 cs;
            angle(a, position(a, tb, tick - tb * ticks), pair, cs.x, cs.y);
            here_angles[i] = cs;
        }
        __syncthreads();                                      // (two sets of angles: nobody is a whole turn ahead)
        float c[N], sn[N];
        if (turns && there) {
            const float4* cs = reinterpret_cast<const float4*>(here_angles + j * half_turn + lane * N);
#pragma unroll
            for (int k = 0; k < N / 2; ++k) {
                const float4 f = cs[k];
                c[2 * k] = f.x; sn[2 * k] = MODE == kForward ? f.y : -f.y;
                c[2 * k + 1] = f.z; sn[2 * k + 1] = MODE == kForward ? f.w : -f.w;
            }
        }
        for (int h = first; h < (heads + share - 1) / share * share; h += share) {
            const bool here = there && h < heads;
            float p[N], q[N], x[N], y[N];
#pragma unroll
            for (int k = 0; k < N; ++k) p[k] = q[k] = x[k] = y[k] = 0.f;
            if (here) {
                if (MODE == kForward || NORM) {
                    from_unit<T>(next[0], x);
                    from_unit<T>(next[1], y);
                }
                if (MODE != kForward) {
                    from_unit<T>(next[2], p);
                    from_unit<T>(next[3], q);
                }
                fetch(h + share);
                if (NORM && s.w && s.w_head) weights(h);
                if (turns && MODE != kForward) turn<INTER, N>(p, q, c, sn);
            }
            if (NORM) {
                float sq = 0.f, m = 0.f;
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    sq = fmaf(x[k], x[k], fmaf(y[k], y[k], sq));
                    if (MODE != kForward) m = fmaf(p[k] * w0[k], x[k], fmaf(q[k] * w1[k], y[k], m));
                }
                for (int o = plan.lanes >> 1; o; o >>= 1) {
                    sq += __shfl_xor_sync(0xffffffffu, sq, o);
                    if (MODE != kForward) m += __shfl_xor_sync(0xffffffffu, m, o);
                }
                const float norm = rsqrtf(fmaf(sq, inverse, a.eps));
                if (MODE == kForward) {
#pragma unroll
                    for (int k = 0; k < N; ++k) x[k] *= norm * w0[k], y[k] *= norm * w1[k];
                } else {
                    const float mean = m * norm * norm * inverse;
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        if (MODE == kBackwardW) {
                            gw0[k] = fmaf(p[k], x[k] * norm, gw0[k]);
                            gw1[k] = fmaf(q[k], y[k] * norm, gw1[k]);
                        }
                        if (MODE == kBackwardEach && here) {
                            sums[h * a.dim + u0 + k] += p[k] * (x[k] * norm);
                            sums[h * a.dim + u1 + k] += q[k] * (y[k] * norm);
                        }
                        p[k] = norm * (p[k] * w0[k] - x[k] * mean);
                        q[k] = norm * (q[k] * w1[k] - y[k] * mean);
                    }
                }
            }
            if (!here) continue;
            if (MODE == kForward) {
                if (turns) turn<INTER, N>(x, y, c, sn);
                store_unit(to + h * to_head + u0, x);
                store_unit(to + h * to_head + u1, y);
            } else {
                store_unit(to + h * to_head + u0, p);
                store_unit(to + h * to_head + u1, q);
            }
        }
    }
    if (MODE == kBackwardW) {
        // the groups' sums in turn: part [block][side][dim]
        float* all = shared;                                  // [groups][dim]
        __syncthreads();
        if (busy) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                all[group * a.dim + u0 + k] = gw0[k];
                all[group * a.dim + u1 + k] = gw1[k];
            }
        }
        __syncthreads();
        for (int i = tid; i < a.dim; i += 256) {
            float sum = 0.f;
            for (int g = 0; g < groups; ++g) sum += all[g * a.dim + i];
            part[((long long)blockIdx.x * 2 + blockIdx.y) * a.dim + i] = sum;
        }
    }
    if (MODE == kBackwardEach) {                              // part [block][queries' heads, keys' heads][dim]
        __syncthreads();
        float* to = part + ((long long)blockIdx.x * (a.s[0].heads + a.s[1].heads) + (blockIdx.y ? a.s[0].heads : 0)) * a.dim;
        for (int i = tid; i < heads * a.dim; i += 256) to[i] = sums[i];
    }
}

constexpr int kSplits = 148 * 2;                             // blocks with sums of their own, at most

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
    need(!g->norm || g->eps > 0, "fg_norm_rotate: eps must be positive");
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

long long work_bytes(const fg_rotate_args* g) {
    if (!g->norm || (!g->gw[0] && !g->gw[1])) return 0;
    const long long sets = std::max<long long>(2, g->w_head[0] || g->w_head[1] ? g->heads[0] + g->heads[1] : 2);
    const long long blocks = std::max<long long>(1, std::min<long long>(kSplits, g->batch * g->ticks));
    return (rows_of(g) + 3) / 4 * 16 + sets * g->dim * blocks * 4;
}

unsigned blocks_for(long long rows) {
    return (unsigned)std::max<long long>(1, std::min<long long>((rows + kWarps - 1) / kWarps, 1 << 20));
}

bool aligned(const void* p, const long long (&st)[3], long long unit) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] % unit == 0 && st[1] % unit == 0 && st[2] % unit == 0;
}
// whether rows are whole pairs of 16-byte units
bool has_units(const Rotate& a, int size, bool backward) {
    const int unit = 16 / size;
    if (a.dim % (2 * unit) || a.turned % (2 * unit) || a.dim / (2 * unit) > 32 || a.batch * a.ticks >= (1ll << 30)) return false;
    for (const Side& s : a.s) {
        if (!s.heads) continue;
        if ((!backward || a.norm) && !aligned(s.x, s.xs, unit)) return false;
        if (backward ? !aligned(s.gy, s.gys, unit) || !aligned(s.gx, s.gxs, unit) : !aligned(s.y, s.ys, unit)) return false;
        if (s.w && (reinterpret_cast<uintptr_t>(s.w) % 16 || s.w_head % 4)) return false;
    }
    return true;
}
template <class T, bool INTER, bool NORM, int MODE>
void launch_units(const Rotate& a, float* part, int& blocks, cudaStream_t st) {
    const int items = a.dim / (2 * Unit<T>::n), half = a.turned / 2, total = (int)(a.batch * a.ticks);
    UnitPlan plan{{1, 1}, 1};
    while (plan.lanes < items) plan.lanes *= 2;
    const int groups = 256 / plan.lanes;
    size_t bytes = 0;
    blocks = 1;
    for (int i = 0; i < 2; ++i) {
        const int heads = a.s[i].heads;
        // as many ticks as leave a group a head or two of one, unless there are too few to go round
        int per = 1;
        while (MODE != kBackwardEach && per < kTicksMost && per * 2 <= groups && groups / per > std::max(1, heads / 2)) per *= 2;
        while (per > 1 && (total + per - 1) / per < 148 * 4) per /= 2;
        plan.per[i] = per;
        bytes = std::max(bytes, (size_t)per * half * 16 + (MODE == kBackwardEach ? (size_t)heads * a.dim * 4 : 0));
        if (heads) blocks = std::max(blocks, (total + per - 1) / per);
    }
    if (MODE == kBackwardW) bytes = std::max(bytes, (size_t)groups * a.dim * 4);
    auto* k = k_rotate_units<T, INTER, NORM, MODE>;
    if (bytes > 48 * 1024) MCK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    blocks = std::min(blocks, MODE >= kBackwardW ? kSplits : 148 * 32);
    k<<<dim3(blocks, a.s[1].heads ? 2 : 1), 256, bytes, st>>>(a, plan, part);
    MCK(cudaGetLastError());
}
template <class T, int MODE>
void launch_units(const Rotate& a, float* part, int& blocks, cudaStream_t st) {
    constexpr bool with_norm = MODE >= kBackwardW;            // (sums of gw are the norm's)
    if (a.norm) a.interleaved ? launch_units<T, true, true, MODE>(a, part, blocks, st) : launch_units<T, false, true, MODE>(a, part, blocks, st);
    else if constexpr (!with_norm) a.interleaved ? launch_units<T, true, false, MODE>(a, part, blocks, st) : launch_units<T, false, false, MODE>(a, part, blocks, st);
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
            int blocks = 0;
            if (has_units(a, sizeof(T), false)) launch_units<T, kForward>(a, nullptr, blocks, st);
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
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            float* part = norms ? norms + (rows + 3) / 4 * 4 : nullptr;
            // (the sums of one set of weights for some heads and sets of their own for others go the general way)
            const bool each = g->w_head[0] || g->w_head[1];
            const bool all_each = (!a.s[0].gw || !a.s[0].heads || g->w_head[0]) && (!a.s[1].gw || !a.s[1].heads || g->w_head[1]);
            const bool fits = !each || (all_each && (g->heads[0] + g->heads[1]) * g->dim * 4 <= 64 * 1024);
            if (rows && has_units(a, sizeof(T), true) && (!norms || fits)) {
                int blocks = 0;
                if (!norms) launch_units<T, kBackward>(a, nullptr, blocks, st);
                else if (each) launch_units<T, kBackwardEach>(a, part, blocks, st);
                else launch_units<T, kBackwardW>(a, part, blocks, st);
                if (norms) {
                    const int n[2] = {(int)sets_of(g, 0) * a.dim, (int)sets_of(g, 1) * a.dim};
                    const int stride = each ? (a.s[0].heads + a.s[1].heads) * a.dim : 2 * a.dim;
                    k_rotate_gw_sum<<<(stride + 31) / 32, 1024, 0, st>>>(part, a.s[0].heads ? a.s[0].gw : nullptr, n[0],
                                                                         a.s[1].heads ? a.s[1].gw : nullptr,
                                                                         each ? a.s[0].heads * a.dim : a.dim, n[1], stride, blocks);
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
                k_rotate_gw_sum<<<(n + 31) / 32, 1024, 0, st>>>(part, a.s[i].gw, n, nullptr, 0, 0, n, splits);
                MCK(cudaGetLastError());
            }
        });
        return 0;
    });
}

}  // extern "C"
