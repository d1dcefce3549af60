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
// gw = the splits' sums added in order
__global__ void k_rotate_gw_sum(const float* __restrict__ part, float* __restrict__ gw, int n, int splits) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += part[(long long)k * n + i];
    gw[i] = s;
}

constexpr int kSplits = 256;

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
    const long long sets = std::max(sets_of(g, 0), sets_of(g, 1));
    return (rows_of(g) + 3) / 4 * 16 + sets * g->dim * kSplits * 4;
}

unsigned blocks_for(long long rows) {
    return (unsigned)std::max<long long>(1, std::min<long long>((rows + kWarps - 1) / kWarps, 1 << 20));
}

}  // namespace

extern "C" {

int fg_norm_rotate(const fg_rotate_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        const Rotate a = checked(g, false);
        const long long rows = rows_of(g);
        if (!rows) return 0;
        by_type(g->type, [&](auto t) {
            k_rotate_any<decltype(t)><<<blocks_for(rows), 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(a, rows);
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
            if (rows) k_rotate_bwd_any<T><<<blocks_for(rows), 32 * kWarps, 0, st>>>(a, rows, norms);
            MCK(cudaGetLastError());
            for (int i = 0; i < 2; ++i) {
                if (!a.s[i].gw || !a.s[i].heads) continue;
                const int sets = (int)sets_of(g, i), n = sets * a.dim;
                need(sets <= 65535, "fg_norm_rotate_bwd: too many heads with weights of their own");
                float* part = norms + (rows + 3) / 4 * 4;
                const int splits = (int)std::max<long long>(1, std::min<long long>(kSplits, g->batch * g->ticks));
                const dim3 grid((a.dim + 127) / 128, sets, splits);
                k_rotate_gw_any<T><<<grid, 128, 0, st>>>(a, i, norms, part, sets, splits);
                k_rotate_gw_sum<<<(n + 127) / 128, 128, 0, st>>>(part, a.s[i].gw, n, splits);
                MCK(cudaGetLastError());
            }
        });
        return 0;
    });
}

}  // extern "C"
