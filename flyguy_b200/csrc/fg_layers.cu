// The layers around a memory: layer norm with its gradients, and dropout by a counter-based generator.
//
//   d = x - mean(x), r = 1 / sqrt(mean(d^2) + eps), y = d r w + b                                         (rows of dim values)
//   g = gy w, gx = r (g - mean(g) - d r mean(g d r)), gw = sum over rows of gy d r, gb = sum over rows of gy
//
//   y = add + (kept ? x / (1 - p) : 0)                                                                    (gx: the same of gy)
//
// A row stays in registers between its statistics (the mean, then the squares of what is left: two sums, so that a mean far
// from zero costs no digits) and its result, so x is read once. The mask is made anew wherever it is needed.
#include "fg_memory.cuh"

namespace {
using namespace fgm;

// V values of T: 16 bytes, or one
template <class T, int V>
__device__ __forceinline__ void load(const T* p, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = to_f(*p);
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_f(e[i]);
    }
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&x)[V]) {
    if constexpr (V == 1) {
        *p = from_f<T>(x[0]);
    } else {
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = from_f<T>(x[i]);
        *reinterpret_cast<uint4*>(p) = u;
    }
}

struct Norm {
    const char *x, *gy;
    char *y, *gx;
    const float *w, *b;
    float* part;                     // [blocks][2][dim]: sums of gy d r and of gy over a block's rows
    long long rows, x_row, gy_row;   // y and gx lie row after row
    int dim;
    float eps;
};

// sums over the threads that share a row: a warp, or the block
template <bool WARP, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* room, int& turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = warp_sum(s[i]);
    if constexpr (!WARP) {
        float* at = room + (turn ^= 1) * 32 * N;              // (two places in turn: one barrier a sum)
        const int warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) at[(threadIdx.x >> 5) * N + i] = s[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = 0.f;
        for (int k = 0; k < warps; ++k) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] += at[k * N + i];
        }
    }
}

// A row's PER units of V values in this thread as d = x - mean (0 past the row's end); r
template <class T, int V, int PER, bool WARP>
__device__ __forceinline__ float centred(const Norm& a, const T* p, int me, int step, float (&d)[PER][V], float* room, int& turn) {
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int c = (me + j * step) * V;
        if (c < a.dim) load<T, V>(p + c, d[j]);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if ((me + j * step) * V < a.dim) {
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += d[j][i];
        }
    }
    row_sums<WARP, 1>(s, room, turn);
    const float mean = s[0] / (float)a.dim;
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const bool in = (me + j * step) * V < a.dim;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            d[j][i] = in ? d[j][i] - mean : 0.f;
            s[0] = fmaf(d[j][i], d[j][i], s[0]);
        }
    }
    row_sums<WARP, 1>(s, room, turn);
    return 1.f / sqrtf(s[0] / (float)a.dim + a.eps);
}

template <class T, int V, int PER, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) k_norm(const __grid_constant__ Norm a) {
    __shared__ float room[64];
    int turn = 0;
    const int me = WARP ? threadIdx.x & 31 : threadIdx.x, step = WARP ? 32 : blockDim.x;
    const long long row = WARP ? blockIdx.x * (long long)(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    float d[PER][V];
    const float r = centred<T, V, PER, WARP>(a, reinterpret_cast<const T*>(a.x) + row * a.x_row, me, step, d, room, turn);
    T* y = reinterpret_cast<T*>(a.y) + row * a.dim;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int c = (me + j * step) * V;
        if (c >= a.dim) continue;
        float w[V], o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = a.w ? a.w[c + i] : 1.f;
            o[i] = a.b ? a.b[c + i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = fmaf(d[j][i] * r, w[i], o[i]);
        store<T, V>(y + c, o);
    }
}

// gx of rows, and this block's sums for gw and gb
template <class T, int V, int PER, bool WARP, bool SUMS>
__global__ void __launch_bounds__(WARP ? 256 : 1024) k_norm_bwd(const __grid_constant__ Norm a) {
    __shared__ float room[128];
    extern __shared__ float sums[];                           // WARP: [warps][32 V] of one unit column
    int turn = 0;
    const int me = WARP ? threadIdx.x & 31 : threadIdx.x, step = WARP ? 32 : blockDim.x;
    const int group = WARP ? threadIdx.x >> 5 : 0, groups = WARP ? blockDim.x >> 5 : 1;
    float aw[SUMS ? PER : 1][V], ab[SUMS ? PER : 1][V];
    if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) aw[j][i] = ab[j][i] = 0.f;
    }
    for (long long row = blockIdx.x * (long long)groups + group; row < a.rows; row += gridDim.x * (long long)groups) {
        float d[PER][V], g[PER][V];
        const T* gy = reinterpret_cast<const T*>(a.gy) + row * a.gy_row;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = (me + j * step) * V;
            if (c < a.dim) load<T, V>(gy + c, g[j]);
        }
        const float r = centred<T, V, PER, WARP>(a, reinterpret_cast<const T*>(a.x) + row * a.x_row, me, step, d, room, turn);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = (me + j * step) * V;
            const bool in = c < a.dim;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                d[j][i] *= r;
                if (!in) g[j][i] = 0.f;
                if constexpr (SUMS) {
                    aw[j][i] = fmaf(g[j][i], d[j][i], aw[j][i]);
                    ab[j][i] += g[j][i];
                }
                if (a.w) g[j][i] *= in ? a.w[c + i] : 0.f;
                s[0] += g[j][i];
                s[1] = fmaf(g[j][i], d[j][i], s[1]);
            }
        }
        row_sums<WARP, 2>(s, room, turn);
        const float m = s[0] / (float)a.dim, k = s[1] / (float)a.dim;
        T* gx = reinterpret_cast<T*>(a.gx) + row * a.dim;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = (me + j * step) * V;
            if (c >= a.dim) continue;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = r * (g[j][i] - m - d[j][i] * k);
            store<T, V>(gx + c, o);
        }
    }
    if constexpr (SUMS) {
        float* part = a.part + (long long)blockIdx.x * 2 * a.dim;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = (me + j * step) * V;
            if constexpr (!WARP) {
                if (c < a.dim) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        part[c + i] = aw[j][i];
                        part[a.dim + c + i] = ab[j][i];
                    }
                }
            } else {
#pragma unroll
                for (int which = 0; which < 2; ++which) {     // the warps' sums in order
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < V; ++i) sums[group * 32 * V + me * V + i] = which ? ab[j][i] : aw[j][i];
                    __syncthreads();
                    for (int e = threadIdx.x; e < 32 * V; e += blockDim.x) {
                        float t = 0.f;
                        for (int k = 0; k < groups; ++k) t += sums[k * 32 * V + e];
                        const int at = j * 32 * V + e;
                        if (at < a.dim) part[which * a.dim + at] = t;
                    }
                }
            }
        }
    }
}

// Rows of any length: read three times, the second and third from the caches.
template <class T>
__global__ void __launch_bounds__(512) k_norm_any(const __grid_constant__ Norm a, float* stats) {
    __shared__ float room[128];
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_row;
        float s[1] = {0.f};
        for (int c = threadIdx.x; c < a.dim; c += 512) s[0] += to_f(x[c]);
        row_sums<false, 1>(s, room, turn);
        const float mean = s[0] / (float)a.dim;
        s[0] = 0.f;
        for (int c = threadIdx.x; c < a.dim; c += 512) {
            const float d = to_f(x[c]) - mean;
            s[0] = fmaf(d, d, s[0]);
        }
        row_sums<false, 1>(s, room, turn);
        const float r = 1.f / sqrtf(s[0] / (float)a.dim + a.eps);
        if (!a.gy) {
            T* y = reinterpret_cast<T*>(a.y) + row * a.dim;
            for (int c = threadIdx.x; c < a.dim; c += 512)
                y[c] = from_f<T>(fmaf((to_f(x[c]) - mean) * r, a.w ? a.w[c] : 1.f, a.b ? a.b[c] : 0.f));
            continue;
        }
        const T* gy = reinterpret_cast<const T*>(a.gy) + row * a.gy_row;
        float t[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < a.dim; c += 512) {
            const float g = to_f(gy[c]) * (a.w ? a.w[c] : 1.f);
            t[0] += g;
            t[1] = fmaf(g, (to_f(x[c]) - mean) * r, t[1]);
        }
        row_sums<false, 2>(t, room, turn);
        const float m = t[0] / (float)a.dim, k = t[1] / (float)a.dim;
        T* gx = reinterpret_cast<T*>(a.gx) + row * a.dim;
        for (int c = threadIdx.x; c < a.dim; c += 512)
            gx[c] = from_f<T>(r * (to_f(gy[c]) * (a.w ? a.w[c] : 1.f) - m - (to_f(x[c]) - mean) * r * k));
        if (stats && threadIdx.x == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = r;
        }
    }
}
// the sums for gw and gb of rows first, first + parts, ..: a thread a column
template <class T>
__global__ void __launch_bounds__(256) k_norm_columns(const __grid_constant__ Norm a, const float* stats) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.dim) return;
    float sw = 0.f, sb = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = to_f(reinterpret_cast<const T*>(a.gy)[row * a.gy_row + c]);
        const float d = to_f(reinterpret_cast<const T*>(a.x)[row * a.x_row + c]) - stats[2 * row];
        sw = fmaf(g, d * stats[2 * row + 1], sw);
        sb += g;
    }
    float* part = a.part + (long long)blockIdx.y * 2 * a.dim;
    part[c] = sw;
    part[a.dim + c] = sb;
}

// gw and gb: the blocks' sums added in a fixed order, 32 columns a block, its 16 warps every 16th of them
__global__ void __launch_bounds__(512) k_norm_sums(const float* __restrict__ part, int blocks, int dim, float* gw, float* gb) {
    __shared__ float s[16][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float* to = blockIdx.y ? gb : gw;
    if (!to) return;
    float t = 0.f;
    if (c < dim)
        for (int k = w; k < blocks; k += 16) t += part[(2ll * k + blockIdx.y) * dim + c];
    s[w][lane] = t;
    __syncthreads();
    if (w == 0 && c < dim) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += s[k][lane];
        to[c] = sum;
    }
}

constexpr int kNormBlocks = 4 * kSms;                         // partial sums of a backward pass at most
constexpr int kLongest = 16384;                               // values of a row that the registers of a block hold

int vector_of(const fg_norm_args* g, bool backward) {
    const int v = g->type == FG_F32 ? 4 : 8;
    const auto fits = [&](const void* p, long long row) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % v == 0; };
    return g->dim % v == 0 && fits(g->x, g->x_row) && (backward ? fits(g->gy, g->gy_row) && fits(g->gx, 0) : fits(g->y, 0)) ? v : 1;
}
Norm norm_of(const fg_norm_args* g) {
    Norm a{};
    a.x = static_cast<const char*>(g->x);
    a.y = static_cast<char*>(g->y);
    a.gy = static_cast<const char*>(g->gy);
    a.gx = static_cast<char*>(g->gx);
    a.w = g->w;
    a.b = g->b;
    a.part = static_cast<float*>(g->work);
    a.rows = g->rows;
    a.x_row = g->x_row;
    a.gy_row = g->gy_row;
    a.dim = (int)g->dim;
    a.eps = (float)g->eps;
    return a;
}
void check(const fg_norm_args* g, const char* who) {
    const std::string w = who;
    if (!g) throw MemErr{w + ": no arguments"};
    if (g->rows < 0 || g->rows > (1ll << 40)) throw MemErr{w + ": rows must be 0 to 2^40"};
    if (g->dim < 1 || g->dim > (1ll << 24)) throw MemErr{w + ": dim must be 1 to 2^24"};
    if (g->type < FG_F32 || g->type > FG_F16) throw MemErr{w + ": unknown type"};
    if (!(g->eps > 0)) throw MemErr{w + ": eps must be positive"};
}
bool any_length(const fg_norm_args* g) { return g->dim > kLongest; }
long long norm_work(const fg_norm_args* g) {
    if (!g->gw && !g->gb) return 0;
    return (kNormBlocks * 2 * g->dim + (any_length(g) ? 2 * g->rows : 0)) * 4;
}

// f(vector width, units a thread, whether a warp takes a row) as types, and the threads that share a row
template <class T, class F>
void by_shape(int v, int dim, F&& f) {
    using std::integral_constant;
    using W = std::true_type;
    using B = std::false_type;
    const int units = (dim + v - 1) / v;
    constexpr int wide = 16 / (int)sizeof(T);
    if (v > 1) {
        using V = integral_constant<int, wide>;
        if (units <= 32) f(V(), integral_constant<int, 1>(), W(), 32);
        else if (units <= 64) f(V(), integral_constant<int, 2>(), W(), 32);
        else if (units <= 128) f(V(), integral_constant<int, 4>(), W(), 32);
        else if (units <= 1024) f(V(), integral_constant<int, 1>(), B(), (units + 31) / 32 * 32);
        else f(V(), integral_constant<int, 4>(), B(), (units + 127) / 128 * 32);
    } else {
        using V = integral_constant<int, 1>;
        if (units <= 128) f(V(), integral_constant<int, 4>(), W(), 32);
        else if (units <= 544) f(V(), integral_constant<int, 17>(), W(), 32);
        else if (units <= 4096) f(V(), integral_constant<int, 4>(), B(), (units + 127) / 128 * 32);
        else f(V(), integral_constant<int, 16>(), B(), (units + 511) / 512 * 32);
    }
}

template <class T>
void norm_forward(const fg_norm_args* g, cudaStream_t st) {
    const Norm a = norm_of(g);
    if (any_length(g)) {
        k_norm_any<T><<<(unsigned)std::min<long long>(a.rows, kSms * 4), 512, 0, st>>>(a, nullptr);
        return;
    }
    by_shape<T>(vector_of(g, false), a.dim, [&](auto v, auto per, auto warp, int threads) {
        constexpr bool W = decltype(warp)::value;
        // a warp a row: few rows spread over the SMs
        const int warps = W ? (int)std::min<long long>(8, (a.rows + kSms - 1) / kSms) : 1;
        const long long blocks = (a.rows + warps - 1) / warps;
        need(blocks < (1ll << 31), "fg_layer_norm: too many rows");
        k_norm<T, decltype(v)::value, decltype(per)::value, W><<<(unsigned)blocks, W ? 32 * warps : threads, 0, st>>>(a);
    });
}

template <class T>
void norm_backward(const fg_norm_args* g, cudaStream_t st) {
    Norm a = norm_of(g);
    const bool sums = g->gw || g->gb;
    int blocks = 0;
    if (any_length(g)) {
        float* stats = sums ? a.part + 2ll * kNormBlocks * a.dim : nullptr;
        k_norm_any<T><<<(unsigned)std::min<long long>(a.rows, kSms * 4), 512, 0, st>>>(a, stats);
        MCK(cudaGetLastError());
        if (sums) {
            blocks = (int)std::min<long long>(a.rows, 64);
            k_norm_columns<T><<<dim3((unsigned)((a.dim + 255) / 256), blocks), 256, 0, st>>>(a, stats);
        }
    } else {
        by_shape<T>(vector_of(g, true), a.dim, [&](auto v, auto per, auto warp, int threads) {
            constexpr int V = decltype(v)::value, PER = decltype(per)::value;
            constexpr bool W = decltype(warp)::value;
            const int warps = W ? (int)std::min<long long>(8, (a.rows + kSms - 1) / kSms) : 1;
            blocks = (int)std::min<long long>(kNormBlocks, (a.rows + warps - 1) / warps);
            if (sums) k_norm_bwd<T, V, PER, W, true><<<blocks, W ? 32 * warps : threads, W ? warps * 32 * V * 4 : 0, st>>>(a);
            else k_norm_bwd<T, V, PER, W, false><<<blocks, W ? 32 * warps : threads, 0, st>>>(a);
        });
    }
    MCK(cudaGetLastError());
    if (sums) k_norm_sums<<<dim3((unsigned)((a.dim + 31) / 32), 2), 512, 0, st>>>(a.part, blocks, a.dim, g->gw, g->gb);
}

// ---- dropout ----------------------------------------------------------------------------------------------------------

// Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011):
// 128 random bits from a counter (block, call) and a key (the seed).
__device__ __forceinline__ uint4 philox(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
        c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1, (uint32_t)a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

struct Drop {
    const char *x, *add;
    char* y;
    const long long* seed;           // on the device, or NULL: seed_value
    long long seed_value, call, n;
    uint32_t least;                  // 16 bits of a value at least this: it stays
    float by;
};

// A thread makes one block of the generator, 8 values of 16 bits. Bound by the memory; the generator's 20 wide products and 40
// exclusive ors are some 100 instructions for 8 values.
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) k_dropout(const __grid_constant__ Drop a) {
    const uint64_t seed = (uint64_t)(a.seed ? *a.seed : a.seed_value);
    for (long long block = blockIdx.x * 256ll + threadIdx.x; block * 8 < a.n; block += gridDim.x * 256ll) {
        const uint4 r = philox(make_uint4((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)a.call, (uint32_t)(a.call >> 32)),
                               (uint32_t)seed, (uint32_t)(seed >> 32));
        const uint32_t bits[8] = {r.x & 0xffff, r.x >> 16, r.y & 0xffff, r.y >> 16, r.z & 0xffff, r.z >> 16, r.w & 0xffff, r.w >> 16};
        const T* x = reinterpret_cast<const T*>(a.x) + block * 8;
        const T* add = a.add ? reinterpret_cast<const T*>(a.add) + block * 8 : nullptr;
        T* y = reinterpret_cast<T*>(a.y) + block * 8;
        constexpr int V = 16 / (int)sizeof(T);
        if (WIDE && block * 8 + 8 <= a.n) {
#pragma unroll
            for (int u = 0; u < 8; u += V) {
                float v[V], o[V];
                load<T, V>(x + u, v);
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = 0.f;
                if (add) load<T, V>(add + u, o);
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = bits[u + i] >= a.least ? fmaf(v[i], a.by, o[i]) : o[i];
                store<T, V>(y + u, o);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (block * 8 + i >= a.n) break;
                const float o = add ? to_f(add[i]) : 0.f;
                y[i] = from_f<T>(bits[i] >= a.least ? fmaf(to_f(x[i]), a.by, o) : o);
            }
        }
    }
}

}  // namespace

extern "C" {

long long fg_layer_norm_work(const fg_norm_args* g) {
    return mem_guard([&]() -> long long {
        check(g, "fg_layer_norm_work");
        return norm_work(g);
    });
}

int fg_layer_norm(const fg_norm_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, "fg_layer_norm");
        if (!g->rows) return 0;
        need(g->x && g->y, "fg_layer_norm: null pointer");
        fg_norm_args f = *g;
        f.gy = nullptr;
        by_type(g->type, [&](auto t) { norm_forward<decltype(t)>(&f, static_cast<cudaStream_t>(stream)); });
        MCK(cudaGetLastError());
        return 0;
    });
}

int fg_layer_norm_bwd(const fg_norm_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, "fg_layer_norm_bwd");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (!g->rows) {                                       // sums of nothing
            if (g->gw) MCK(cudaMemsetAsync(g->gw, 0, g->dim * 4, st));
            if (g->gb) MCK(cudaMemsetAsync(g->gb, 0, g->dim * 4, st));
            return 0;
        }
        need(g->x && g->gy && g->gx, "fg_layer_norm_bwd: null pointer");
        const long long bytes = norm_work(g);
        need(!bytes || (g->work && g->work_bytes >= bytes), "fg_layer_norm_bwd: the workspace is too small");
        need(reinterpret_cast<uintptr_t>(g->work) % 16 == 0, "fg_layer_norm_bwd: the workspace is not 16-byte aligned");
        by_type(g->type, [&](auto t) { norm_backward<decltype(t)>(g, st); });
        MCK(cudaGetLastError());
        return 0;
    });
}

int fg_dropout(const fg_dropout_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        need(g, "fg_dropout: no arguments");
        need(g->n >= 0 && g->n <= (1ll << 46), "fg_dropout: n must be 0 to 2^46");
        need(g->least >= 0 && g->least < 65536, "fg_dropout: least must be 0 to 65535");
        need(g->type >= FG_F32 && g->type <= FG_F16, "fg_dropout: unknown type");
        if (!g->n) return 0;
        need(g->x && g->y, "fg_dropout: null pointer");
        Drop a{};
        a.x = static_cast<const char*>(g->x);
        a.add = static_cast<const char*>(g->add);
        a.y = static_cast<char*>(g->y);
        a.seed = g->seed;
        a.seed_value = g->seed_value;
        a.call = g->call;
        a.n = g->n;
        a.least = (uint32_t)g->least;
        a.by = (float)(65536.0 / (65536.0 - (double)g->least));
        const auto at16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
        const bool wide = at16(a.x) && at16(a.add) && at16(a.y);
        const unsigned blocks = (unsigned)std::min<long long>((a.n + 2047) / 2048, kSms * 64);
        by_type(g->type, [&](auto t) {
            auto* kernel = wide ? k_dropout<decltype(t), true> : k_dropout<decltype(t), false>;
            kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
        });
        MCK(cudaGetLastError());
        return 0;
    });
}

}  // extern "C"
