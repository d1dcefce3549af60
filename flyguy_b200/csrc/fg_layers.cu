// The layers around a memory: layer norm with its gradients, and dropout by a counter-based generator.
//
//   d = x - mean(x), r = 1 / sqrt(mean(d^2) + eps), y = d r w + b                                         (rows of dim values)
//   g = gy w, gx = r (g - mean(g) - d r mean(g d r)), gw = sum over rows of gy d r, gb = sum over rows of gy
//
//   y = add + (kept ? x / (1 - p) : 0)                                                                    (gx: the same of gy)
//
// A row stays on the chip between its statistics and its result, so x is read once. The statistics are the mean m, as good as fp32 sums
// make it, and then of d = x - m the sum, for what m lacks, and the squares: d r = (x - m) r - mean(d) r, var = mean(d^2) - mean(d)^2, so
// that a mean far from zero costs no digits. The mask is made anew wherever it is needed.
#include "fg_memory.cuh"

namespace {
using namespace fgm;

// V values of T as they lie in memory: 16 bytes, or one value
template <class T, int V>
struct alignas(V > 1 ? 16 : sizeof(T)) Unit {
    T v[V];
};
template <class T, int V>
__device__ __forceinline__ Unit<T, V> load(const T* p) {
    return *reinterpret_cast<const Unit<T, V>*>(p);
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&x)[V]) {
    Unit<T, V> u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.v[i] = from_f<T>(x[i]);
    *reinterpret_cast<Unit<T, V>*>(p) = u;
}
// V values of the weight or the bias (aligned where V is over 1; NULL: `other`)
template <int V>
__device__ __forceinline__ void load_w(const float* p, int c, float other, float (&w)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = other;
    if (!p) return;
    if constexpr (V == 1) {
        w[0] = p[c];
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(w + i) = *reinterpret_cast<const float4*>(p + c + i);
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

// sums over the threads that share a row: GROUP lanes, or (0) the block, which hands them over in two places of `room` in turn, each of WIDEST
// sums of 16 warps, the most that the kernel asks for at once. (One barrier a sum: a place is written again only after the barrier of the sum
// between, and that holds for sums of unequal numbers because the places are the kernel's and not the sum's.)
template <int GROUP, int WIDEST, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* room, int& turn) {
    static_assert(N <= WIDEST, "a place holds the sums");
#pragma unroll
    for (int o = (GROUP ? GROUP : 32) / 2; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    if constexpr (GROUP == 0) {
        float* at = room + (turn ^= 1) * 16 * WIDEST;
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

// from the means of d and of d^2
__device__ __forceinline__ void deviation(float mean, float square, float eps, float& inv, float& lack) {
    inv = 1.f / sqrtf(fmaxf(fmaf(-mean, mean, square), 0.f) + eps);
    lack = -mean * inv;
}

// What a thread has of ROWS rows: PER units of V values of each, kept as they came so that 16-bit values take half the registers
template <class T, int V, int PER, int GROUP, int ROWS>
struct Rows {
    Unit<T, V> u[ROWS][PER];
    int me, step;
    __device__ __forceinline__ int column(int j) const { return (me + j * step) * V; }
    __device__ __forceinline__ void fetch(const char* p, long long row, long long rows, long long stride, int dim) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (row + r < rows && column(j) < dim) u[r][j] = load<T, V>(reinterpret_cast<const T*>(p) + (row + r) * stride + column(j));
    }
    // the values d r are (x - mean) inv + lack; rows past the last are worked on as they are
    __device__ __forceinline__ void stats(int dim, float eps, float (&mean)[ROWS], float (&inv)[ROWS], float (&lack)[ROWS], float* room, int& turn) const {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            mean[r] = 0.f;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (column(j) < dim) {
#pragma unroll
                    for (int i = 0; i < V; ++i) mean[r] += to_f(u[r][j].v[i]);
                }
        }
        row_sums<GROUP, 2 * ROWS>(mean, room, turn);
        float s[2 * ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            mean[r] /= (float)dim;
            s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (column(j) < dim) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = to_f(u[r][j].v[i]) - mean[r];
                        s[2 * r] += d;
                        s[2 * r + 1] = fmaf(d, d, s[2 * r + 1]);
                    }
                }
        }
        row_sums<GROUP, 2 * ROWS>(s, room, turn);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) deviation(s[2 * r] / (float)dim, s[2 * r + 1] / (float)dim, eps, inv[r], lack[r]);
    }
};

template <class T, int V, int PER, int GROUP, int ROWS>
__global__ void __launch_bounds__(GROUP ? 256 : 512) k_norm(const __grid_constant__ Norm a) {
    __shared__ float room[64 * ROWS];
    int turn = 0;
    Rows<T, V, PER, GROUP, ROWS> x;
    x.me = GROUP ? threadIdx.x % (GROUP ? GROUP : 1) : threadIdx.x;
    x.step = GROUP ? GROUP : blockDim.x;
    const long long row = (GROUP ? blockIdx.x * (long long)(blockDim.x / (GROUP ? GROUP : 1)) + threadIdx.x / (GROUP ? GROUP : 1) : blockIdx.x) * ROWS;
    x.fetch(a.x, row, a.rows, a.x_row, a.dim);
    float mean[ROWS], inv[ROWS], lack[ROWS];
    x.stats(a.dim, a.eps, mean, inv, lack, room, turn);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int c = x.column(j);
        if (c >= a.dim) continue;
        float w[V], b[V];
        load_w<V>(a.w, c, 1.f, w);
        load_w<V>(a.b, c, 0.f, b);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (row + r >= a.rows) break;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(fmaf(to_f(x.u[r][j].v[i]) - mean[r], inv[r], lack[r]), w[i], b[i]);
            store<T, V>(reinterpret_cast<T*>(a.y) + (row + r) * a.dim + c, o);
        }
    }
}

// gx of rows, and this block's sums for gw and gb. While a group of rows is worked on the next one is on its way.
template <class T, int V, int PER, int GROUP, int ROWS, bool SUMS>
__global__ void __launch_bounds__(GROUP ? 128 : 512, GROUP ? 3 : 1) k_norm_bwd(const __grid_constant__ Norm a) {
    __shared__ float room[64 * ROWS];
    extern __shared__ float sums[];                           // GROUP: [groups][GROUP V] of one unit column
    constexpr int kGroup = GROUP ? GROUP : 1;
    int turn = 0;
    const int group = GROUP ? threadIdx.x / kGroup : 0, groups = GROUP ? blockDim.x / kGroup : 1;
    Rows<T, V, PER, GROUP, ROWS> x, g, next_x, next_g;
    x.me = g.me = next_x.me = next_g.me = GROUP ? threadIdx.x % kGroup : threadIdx.x;
    x.step = g.step = next_x.step = next_g.step = GROUP ? GROUP : blockDim.x;
    float aw[SUMS ? PER : 1][V], ab[SUMS ? PER : 1][V];
    if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) aw[j][i] = ab[j][i] = 0.f;
    }
    const long long step = gridDim.x * (long long)groups * ROWS, first = (blockIdx.x * (long long)groups) * ROWS;
    next_x.fetch(a.x, first + group * ROWS, a.rows, a.x_row, a.dim);
    next_g.fetch(a.gy, first + group * ROWS, a.rows, a.gy_row, a.dim);
    for (long long base = first; base < a.rows; base += step) {   // (the block's groups stay together)
        const long long row = base + group * ROWS;
        x = next_x;
        g = next_g;
        next_x.fetch(a.x, row + step, a.rows, a.x_row, a.dim);
        next_g.fetch(a.gy, row + step, a.rows, a.gy_row, a.dim);
        float mean[ROWS], inv[ROWS], lack[ROWS], s[2 * ROWS];
        x.stats(a.dim, a.eps, mean, inv, lack, room, turn);
#pragma unroll
        for (int r = 0; r < 2 * ROWS; ++r) s[r] = 0.f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = x.column(j);
            if (c >= a.dim) continue;
            float w[V];
            load_w<V>(a.w, c, 1.f, w);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (row + r >= a.rows) break;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = fmaf(to_f(x.u[r][j].v[i]) - mean[r], inv[r], lack[r]), y = to_f(g.u[r][j].v[i]), z = y * w[i];
                    if constexpr (SUMS) {
                        aw[j][i] = fmaf(y, d, aw[j][i]);
                        ab[j][i] += y;
                    }
                    s[2 * r] += z;
                    s[2 * r + 1] = fmaf(z, d, s[2 * r + 1]);
                }
            }
        }
        row_sums<GROUP, 2 * ROWS>(s, room, turn);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = x.column(j);
            if (c >= a.dim) continue;
            float w[V];
            load_w<V>(a.w, c, 1.f, w);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (row + r >= a.rows) break;
                const float m = s[2 * r] / (float)a.dim, k = s[2 * r + 1] / (float)a.dim;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i)
                    o[i] = inv[r] * (to_f(g.u[r][j].v[i]) * w[i] - m - fmaf(to_f(x.u[r][j].v[i]) - mean[r], inv[r], lack[r]) * k);
                store<T, V>(reinterpret_cast<T*>(a.gx) + (row + r) * a.dim + c, o);
            }
        }
    }
    if constexpr (SUMS) {
        float* part = a.part + (long long)blockIdx.x * 2 * a.dim;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = x.column(j);
            if constexpr (GROUP == 0) {
                if (c < a.dim) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        part[c + i] = aw[j][i];
                        part[a.dim + c + i] = ab[j][i];
                    }
                }
            } else {
#pragma unroll
                for (int which = 0; which < 2; ++which) {     // the groups' sums in order
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < V; ++i) sums[(group * GROUP + x.me) * V + i] = which ? ab[j][i] : aw[j][i];
                    __syncthreads();
                    for (int e = threadIdx.x; e < GROUP * V; e += blockDim.x) {
                        float t = 0.f;
                        for (int k = 0; k < groups; ++k) t += sums[k * GROUP * V + e];
                        const int at = j * GROUP * V + e;
                        if (at < a.dim) part[which * a.dim + at] = t;
                    }
                }
            }
        }
    }
}

// Many rows, a warp each, that copy themselves ahead: a lane's units of the next DEPTH - 1 rows are on their way to places in shared
// memory that it alone reads, so that nothing but its own copies is waited for. With the rows in shared memory (read again for each
// step) the registers are the sums', 16 warps share an SM and 16 x DEPTH rows are in flight.
// SHIFT: rows that begin anywhere, at the same place in 16 bytes in x, gy and what comes out. A warp takes every so many-th row, a multiple of
// 8, so its rows all begin alike; its first and last units reach into the neighbours, whose values count for nothing.
template <class T, int V, bool BACK>
struct Ring {
    static constexpr int depth = BACK ? 3 : 4, warps = 4, tensors = BACK ? 2 : 1;
    static int units(int dim, bool shift) { return (dim + (shift ? V - 1 : 0) + V - 1) / V; }
    // rows' places, in rounds of 32 units, and the weight, with a shift as each warp reads it
    static int bytes(int rounds, bool shift) { return (depth * tensors * 512 * warps + (BACK ? 128 * V * (shift ? warps : 1) : 0)) * rounds; }
};
__device__ __forceinline__ void copy_ahead(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// Values as fp32, in pairs (one instruction for two) where a unit has several
template <int V>
using Lane = std::conditional_t<(V > 1), uint64_t, float>;
template <class P>
__device__ __forceinline__ P same(float x) {
    if constexpr (std::is_same<P, float>::value) return x;
    else return two(x, x);
}
__device__ __forceinline__ float plus(float x, float y) { return x + y; }
__device__ __forceinline__ uint64_t plus(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ float times(float x, float y) { return x * y; }
__device__ __forceinline__ uint64_t times(uint64_t x, uint64_t y) { return mul2(x, y); }
__device__ __forceinline__ float times_plus(float x, float y, float z) { return fmaf(x, y, z); }
__device__ __forceinline__ uint64_t times_plus(uint64_t x, uint64_t y, uint64_t z) { return fma2(x, y, z); }
__device__ __forceinline__ float both(float x) { return x; }
__device__ __forceinline__ float both(uint64_t x) { return sum2(x); }
template <class T, int V>
__device__ __forceinline__ Lane<V> lane_of(const Unit<T, V>& u, int i) {
    if constexpr (V == 1) return to_f(u.v[0]);
    else return two(to_f(u.v[2 * i]), to_f(u.v[2 * i + 1]));
}
template <int V>
__device__ __forceinline__ Lane<V> lane_of(const float (&w)[V], int i) {
    if constexpr (V == 1) return w[0];
    else return two(w[2 * i], w[2 * i + 1]);
}
template <int V>
__device__ __forceinline__ void values_of(Lane<V> p, int i, float (&v)[V]) {
    if constexpr (V == 1) v[0] = p;
    else halves(p, v[2 * i], v[2 * i + 1]);
}

template <class T, int V, int PER, bool SHIFT, bool BACK, bool SUMS>
__global__ void __launch_bounds__(128, 4) k_norm_ring(const __grid_constant__ Norm a, int rounds) {
    using R = Ring<T, V, BACK>;
    using P = Lane<V>;
    constexpr int N = V / 2;
    extern __shared__ __align__(16) unsigned char ring[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, place_bytes = rounds * 512, stage = R::tensors * place_bytes;
    unsigned char* mine = ring + warp * R::depth * stage + lane * 16;
    const long long step = gridDim.x * (long long)R::warps;
    long long row = blockIdx.x * (long long)R::warps + warp;
    const int shift = SHIFT ? (int)((reinterpret_cast<uintptr_t>(a.x) / sizeof(T) + (unsigned long long)(row * a.x_row)) % V) : 0;
    const auto column = [&](int j) { return (lane + 32 * j) * V - shift; };   // may be up to V - 1 before the row
    const auto edge = [&](int c) { return SHIFT && (c < 0 || c + V > a.dim); };
    const auto inside = [&](int c) { return c >= 0 && c < a.dim; };
    const auto fetch = [&](long long row, int place) {
        if (row < a.rows) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int c = column(j);
                if (c >= a.dim) break;
                unsigned char* to = mine + place * stage + j * 512;
#pragma unroll
                for (int k = 0; k < R::tensors; ++k) {
                    const T* p = reinterpret_cast<const T*>(k ? a.gy : a.x) + row * (k ? a.gy_row : a.x_row) + c;
                    if (SHIFT && c + V > a.dim && row + 1 == a.rows) {   // (nothing is read behind the last row)
                        Unit<T, V> u{};
                        for (int i = 0; i < V; ++i)
                            if (inside(c + i)) u.v[i] = p[i];
                        *reinterpret_cast<Unit<T, V>*>(to + k * place_bytes) = u;
                    } else {
                        copy_ahead((uint32_t)__cvta_generic_to_shared(to + k * place_bytes), p);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // forward the weight and the bias stay in registers; back the sums do, and the weight lies in shared memory as the lanes read it
    P w[BACK ? 1 : PER][N], b[BACK ? 1 : PER][N], aw[SUMS ? PER : 1][N], ab[SUMS ? PER : 1][N];
    float* sw = reinterpret_cast<float*>(ring + R::warps * R::depth * stage) + (SHIFT ? warp * 32 * V * rounds : 0) + lane * 4;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int c = column(j);
        float v[V], o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = a.w && inside(c + i) ? a.w[c + i] : 1.f;
            o[i] = !BACK && a.b && inside(c + i) ? a.b[c + i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (!BACK) {
                w[j][i] = lane_of<V>(v, i);
                b[j][i] = lane_of<V>(o, i);
            }
            if constexpr (SUMS) aw[j][i] = ab[j][i] = same<P>(0.f);
        }
        if (BACK && c < a.dim && (SHIFT || warp == 0)) {
#pragma unroll
            for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(sw + (j * V + i) * 32) = *reinterpret_cast<const float4*>(v + i);
        }
    }
    if (BACK && !SHIFT) __syncthreads();
    const auto weight = [&](int j, P(&to)[N]) {
        float v[V];
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(sw + (j * V + i) * 32);
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = lane_of<V>(v, i);
    };
    // pairs outside the row as zeros
    const auto keep = [&](int c, P(&v)[N]) {
        if (edge(c)) {
            float x[V];
#pragma unroll
            for (int i = 0; i < N; ++i) values_of<V>(v[i], i, x);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!inside(c + i)) x[i] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = lane_of<V>(x, i);
        }
    };
    const auto put = [&](T* p, int c, const float (&o)[V]) {
        if (edge(c)) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (inside(c + i)) p[c + i] = from_f<T>(o[i]);
        } else {
            store<T, V>(p + c, o);
        }
    };
#pragma unroll
    for (int k = 0; k < R::depth - 1; ++k) fetch(row + k * step, k);
    int place = 0;
    for (; row < a.rows; row += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(R::depth - 2) : "memory");
        fetch(row + (R::depth - 1) * step, place ? place - 1 : R::depth - 1);
        const unsigned char* at = mine + place * stage;
        place = place + 1 == R::depth ? 0 : place + 1;
        const auto unit = [&](int j) { return *reinterpret_cast<const Unit<T, V>*>(at + j * 512); };
        const auto gunit = [&](int j) { return *reinterpret_cast<const Unit<T, V>*>(at + place_bytes + j * 512); };
        P sum = same<P>(0.f);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = column(j);
            if (c >= a.dim) break;
            const Unit<T, V> x = unit(j);
            P d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = lane_of<T, V>(x, i);
            keep(c, d);
#pragma unroll
            for (int i = 0; i < N; ++i) sum = plus(sum, d[i]);
        }
        const P off = same<P>(-warp_sum(both(sum)) / (float)a.dim);   // - mean
        P squares = same<P>(0.f), s0 = squares, s1 = squares;
        sum = squares;
        // back: sums of g and g d with them, and g d r = r (g d) + lack g, so that a row is gone over three times
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = column(j);
            if (c >= a.dim) break;
            const Unit<T, V> x = unit(j);
            P d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = plus(lane_of<T, V>(x, i), off);
            keep(c, d);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sum = plus(sum, d[i]);
                squares = times_plus(d[i], d[i], squares);
            }
            if constexpr (BACK) {
                const Unit<T, V> g = gunit(j);
                P y[N], v[N];
                weight(j, v);
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = lane_of<T, V>(g, i);
                keep(c, y);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const P z = times(y[i], v[i]);
                    s0 = plus(s0, z);
                    s1 = times_plus(z, d[i], s1);
                }
            }
        }
        float one, other;
        deviation(warp_sum(both(sum)) / (float)a.dim, warp_sum(both(squares)) / (float)a.dim, a.eps, one, other);
        const P inv = same<P>(one), lack = same<P>(other);
        if constexpr (!BACK) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int c = column(j);
                if (c >= a.dim) break;
                const Unit<T, V> x = unit(j);
                float o[V];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    values_of<V>(times_plus(times_plus(plus(lane_of<T, V>(x, i), off), inv, lack), w[j][i], b[j][i]), i, o);
                put(reinterpret_cast<T*>(a.y) + row * a.dim, c, o);
            }
        } else {
            const float g = warp_sum(both(s0)), gd = warp_sum(both(s1));
            const P m = same<P>(-g / (float)a.dim), k = same<P>(-fmaf(gd, one, g * other) / (float)a.dim);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int c = column(j);
                if (c >= a.dim) break;
                const Unit<T, V> x = unit(j), g = gunit(j);
                P v[N];
                weight(j, v);
                float o[V];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const P h = times_plus(plus(lane_of<T, V>(x, i), off), inv, lack), y = lane_of<T, V>(g, i);
                    if constexpr (SUMS) {                     // (of values outside the row: never used)
                        aw[j][i] = times_plus(y, h, aw[j][i]);
                        ab[j][i] = plus(ab[j][i], y);
                    }
                    values_of<V>(times(times_plus(h, k, times_plus(y, v[i], m)), inv), i, o);
                }
                put(reinterpret_cast<T*>(a.gx) + row * a.dim, c, o);
            }
        }
    }
    if constexpr (SUMS) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        float* part = a.part + (long long)blockIdx.x * 2 * a.dim;
        float* sums = reinterpret_cast<float*>(ring);         // without a shift [warps][32 V] of one round's columns, with one [dim]
        if constexpr (!SHIFT) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    float v[V];
#pragma unroll
                    for (int i = 0; i < N; ++i) values_of<V>(which ? ab[j][i] : aw[j][i], i, v);
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < V; i += 4)
                        *reinterpret_cast<float4*>(sums + threadIdx.x * V + i) = *reinterpret_cast<const float4*>(v + i);
                    __syncthreads();
                    for (int e = threadIdx.x; e < 32 * V; e += 128) {
                        float t = 0.f;
#pragma unroll
                        for (int k = 0; k < R::warps; ++k) t += sums[k * 32 * V + e];
                        const int c = j * 32 * V + e;
                        if (c < a.dim) part[which * a.dim + c] = t;
                    }
                }
            return;
        }
#pragma unroll
        for (int which = 0; which < 2; ++which)
            for (int k = 0; k < R::warps; ++k) {              // one warp after another: the order is fixed
                __syncthreads();
                if (k != warp) continue;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (column(j) >= a.dim) break;
                    float v[V];
#pragma unroll
                    for (int i = 0; i < N; ++i) values_of<V>(which ? ab[j][i] : aw[j][i], i, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int c = column(j) + i;
                        if (!inside(c)) continue;
                        const float t = k ? sums[c] + v[i] : v[i];
                        if (k + 1 < R::warps) sums[c] = t;
                        else part[which * a.dim + c] = t;
                    }
                }
            }
    }
}

// Rows of any length: read three times, the second and third from the caches.
template <class T>
__global__ void __launch_bounds__(512) k_norm_any(const __grid_constant__ Norm a, float* stats) {
    __shared__ float room[64];
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_row;
        float s[1] = {0.f};
        for (int c = threadIdx.x; c < a.dim; c += 512) s[0] += to_f(x[c]);
        row_sums<0, 2>(s, room, turn);
        const float mean = s[0] / (float)a.dim;
        float q[2] = {0.f, 0.f}, r, lack;
        for (int c = threadIdx.x; c < a.dim; c += 512) {
            const float d = to_f(x[c]) - mean;
            q[0] += d;
            q[1] = fmaf(d, d, q[1]);
        }
        row_sums<0, 2>(q, room, turn);
        deviation(q[0] / (float)a.dim, q[1] / (float)a.dim, a.eps, r, lack);
        if (!a.gy) {
            T* y = reinterpret_cast<T*>(a.y) + row * a.dim;
            for (int c = threadIdx.x; c < a.dim; c += 512)
                y[c] = from_f<T>(fmaf(fmaf(to_f(x[c]) - mean, r, lack), a.w ? a.w[c] : 1.f, a.b ? a.b[c] : 0.f));
            continue;
        }
        const T* gy = reinterpret_cast<const T*>(a.gy) + row * a.gy_row;
        float t[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < a.dim; c += 512) {
            const float g = to_f(gy[c]) * (a.w ? a.w[c] : 1.f);
            t[0] += g;
            t[1] = fmaf(g, fmaf(to_f(x[c]) - mean, r, lack), t[1]);
        }
        row_sums<0, 2>(t, room, turn);
        const float m = t[0] / (float)a.dim, k = t[1] / (float)a.dim;
        T* gx = reinterpret_cast<T*>(a.gx) + row * a.dim;
        for (int c = threadIdx.x; c < a.dim; c += 512)
            gx[c] = from_f<T>(r * (to_f(gy[c]) * (a.w ? a.w[c] : 1.f) - m - fmaf(to_f(x[c]) - mean, r, lack) * k));
        if (stats && threadIdx.x == 0) {
            stats[3 * row] = mean;
            stats[3 * row + 1] = r;
            stats[3 * row + 2] = lack;
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
        const float d = to_f(reinterpret_cast<const T*>(a.x)[row * a.x_row + c]) - stats[3 * row];
        sw = fmaf(g, fmaf(d, stats[3 * row + 1], stats[3 * row + 2]), sw);
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
#pragma unroll 8
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

constexpr int kNormBlocks = 12 * kSms;                         // partial sums of a backward pass at most
constexpr int kAnyBlocks = 64;                                // the same of rows of any length
constexpr int kLongest = 8192;                                // values of a row that the registers of a block hold

int vector_of(const fg_norm_args* g, bool backward) {
    const int v = g->type == FG_F32 ? 4 : 8;
    const auto fits = [&](const void* p, long long row) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % v == 0; };
    return g->dim % v == 0 && fits(g->x, g->x_row) && fits(g->w, 0) && fits(g->b, 0) && (backward ? fits(g->gy, g->gy_row) && fits(g->gx, 0) : fits(g->y, 0)) ? v : 1;
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
    if (!((float)g->eps > 0)) throw MemErr{w + ": eps must be positive in fp32"};
}
bool any_length(const fg_norm_args* g) { return g->dim > kLongest; }
// blocks that leave sums for gw and gb, at most
long long norm_blocks(const fg_norm_args* g) { return std::min<long long>(g->rows, any_length(g) ? kAnyBlocks : kNormBlocks); }
long long norm_work(const fg_norm_args* g) {
    if (!g->gw && !g->gb) return 0;
    return (norm_blocks(g) * 2 * g->dim + (any_length(g) ? 3 * g->rows : 0)) * 4;
}

constexpr int kSumThreads = 128;                              // of a backward block whose lanes share rows

// What the ring does not take: few rows, short ones, ones whose tensors begin unlike. f(V, PER, GROUP, rows at once forward and back) as types,
// and the threads that share a row: 8 lanes a short one, a warp up to 64 units, then a block (its barriers cost several rows' sums at once;
// 65,536 rows of 1,024 in bf16 and back took 87 + 207 us this way, 55 + 160 with a warp a row in registers, 54 + 85 in the ring).
template <class T, class F>
void by_shape(int v, int dim, F&& f) {
    const int units = (dim + v - 1) / v;
    constexpr int wide = 16 / (int)sizeof(T);
    const auto is = [](auto x) { return x; };
    using std::integral_constant;
#define SHAPE(V, PER, GROUP, ROWS, BACK, THREADS)                                                                                  \
    f(is(integral_constant<int, V>()), is(integral_constant<int, PER>()), is(integral_constant<int, GROUP>()),                     \
      is(integral_constant<int, ROWS>()), is(integral_constant<int, BACK>()), THREADS)
    const auto block = [&](int per) { return (units + 32 * per - 1) / (32 * per) * 32; };
    if (v > 1) {
        if (units <= 8) SHAPE(wide, 1, 8, 2, 2, 8);
        else if (units <= 16) SHAPE(wide, 2, 8, 1, 1, 8);
        else if (units <= 32) SHAPE(wide, 1, 32, 2, 2, 32);
        else if (units <= 64) SHAPE(wide, 2, 32, 2, 1, 32);
        else if (units <= 512) SHAPE(wide, 1, 0, 4, 2, block(1));
        else SHAPE(wide, 16 / wide, 0, 1, 1, block(16 / wide));
    } else {
        if (units <= 32) SHAPE(1, 4, 8, 1, 1, 8);
        else if (units <= 128) SHAPE(1, 4, 32, 2, 2, 32);
        else if (units <= 2048) SHAPE(1, 4, 0, 4, 2, block(4));
        else SHAPE(1, 16, 0, 1, 1, block(16));
    }
#undef SHAPE
}

// f(PER, SHIFT) as types where rows are many and go through the ring: up to 128 units of 16 bytes, beginning at one place in 16 bytes in
// all that is read and written
template <class T, class F>
bool by_ring(const fg_norm_args* g, bool back, F&& f) {
    constexpr int V = 16 / (int)sizeof(T);
    using std::integral_constant;
    const auto fits = [&](const void* p, long long row) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (row - g->dim) % V == 0; };
    if (g->rows < 16 * kSms || !fits(g->x, g->x_row)) return false;
    if (back ? !fits(g->gy, g->gy_row) || !fits(g->gx, g->dim) : !fits(g->y, g->dim)) return false;
    const bool shift = g->dim % V != 0;
    if (shift && (g->x_row < g->dim || (back && g->gy_row < g->dim))) return false;   // (behind a row lies another)
    const int units = Ring<T, V, false>::units((int)g->dim, shift);
    constexpr int most = 32 / V;                             // 32 values a lane
    if (units <= 16 || units > 32 * most) return false;      // (short rows: several to a warp)
    const auto by_per = [&](auto per) {
        if (shift) f(per, std::true_type());
        else f(per, std::false_type());
    };
    if (units <= 32) by_per(integral_constant<int, 1>());
    else if (units <= 64) by_per(integral_constant<int, 2>());
    else if (units <= 128 || most == 4) by_per(integral_constant<int, 4>());
    else by_per(integral_constant<int, most>());
    return true;
}
// As many as run at once (a second round of them would find the SMs half empty: 137 instead of 89 us), and an even number: 4 rows a
// block, so a warp's rows are a multiple of 8 apart.
template <class T, bool SHIFT, bool BACK>
int ring_blocks(int dim) {
    using R = Ring<T, 16 / (int)sizeof(T), BACK>;
    return kSms * std::min(4, 220 * 1024 / (R::bytes((R::units(dim, SHIFT) + 31) / 32, SHIFT) + 1024));
}
template <class T, int PER, bool SHIFT, bool BACK, bool SUMS>
void ring_launch(const Norm& a, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    using R = Ring<T, V, BACK>;
    auto* kernel = k_norm_ring<T, V, PER, SHIFT, BACK, SUMS>;
    static OnEachDevice here;
    here.first(current_device(), [&] { allow_shared(kernel, R::bytes(PER, SHIFT)); });
    const int rounds = (R::units(a.dim, SHIFT) + 31) / 32;
    kernel<<<ring_blocks<T, SHIFT, BACK>(a.dim), 128, R::bytes(rounds, SHIFT), st>>>(a, rounds);
}

template <class T>
void norm_forward(const fg_norm_args* g, cudaStream_t st) {
    const Norm a = norm_of(g);
    if (any_length(g)) {
        k_norm_any<T><<<(unsigned)std::min<long long>(a.rows, kSms * 4), 512, 0, st>>>(a, nullptr);
        return;
    }
    if (by_ring<T>(g, false, [&](auto per, auto shift) { ring_launch<T, decltype(per)::value, decltype(shift)::value, false, false>(a, st); })) return;
    by_shape<T>(vector_of(g, false), a.dim, [&](auto v, auto per, auto group, auto rows, auto, int threads) {
        constexpr int G = decltype(group)::value, R = decltype(rows)::value;
        // few rows: a warp a block, spread over the SMs
        const int block = G ? a.rows >= 16 * kSms * R ? 256 : 32 : threads;
        const long long at_once = (G ? block / threads : 1) * R, blocks = (a.rows + at_once - 1) / at_once;
        need(blocks < (1ll << 31), "fg_layer_norm: too many rows");
        k_norm<T, decltype(v)::value, decltype(per)::value, G, R><<<(unsigned)blocks, block, 0, st>>>(a);
    });
}

template <class T>
void norm_backward(const fg_norm_args* g, cudaStream_t st) {
    Norm a = norm_of(g);
    const bool sums = g->gw || g->gb;
    int blocks = 0;
    if (any_length(g)) {
        float* stats = sums ? a.part + 2 * norm_blocks(g) * a.dim : nullptr;
        k_norm_any<T><<<(unsigned)std::min<long long>(a.rows, kSms * 4), 512, 0, st>>>(a, stats);
        MCK(cudaGetLastError());
        if (sums) {
            blocks = (int)norm_blocks(g);
            k_norm_columns<T><<<dim3((unsigned)((a.dim + 255) / 256), blocks), 256, 0, st>>>(a, stats);
        }
    } else if (by_ring<T>(g, true, [&](auto per, auto shift) {
                   blocks = ring_blocks<T, decltype(shift)::value, true>(a.dim);
                   if (sums) ring_launch<T, decltype(per)::value, decltype(shift)::value, true, true>(a, st);
                   else ring_launch<T, decltype(per)::value, decltype(shift)::value, true, false>(a, st);
               })) {
    } else {
        by_shape<T>(vector_of(g, true), a.dim, [&](auto v, auto per, auto group, auto, auto rows, int threads) {
            constexpr int V = decltype(v)::value, PER = decltype(per)::value, G = decltype(group)::value, R = decltype(rows)::value;
            const int block = G ? kSumThreads : threads;
            const long long at_once = (G ? block / threads : 1) * R;
            blocks = (int)std::min<long long>(G ? 3 * kSms : std::min(kNormBlocks, kSms * std::max(1, 768 / block)), (a.rows + at_once - 1) / at_once);
            if (sums) k_norm_bwd<T, V, PER, G, R, true><<<blocks, block, G ? block * V * 4 : 0, st>>>(a);
            else k_norm_bwd<T, V, PER, G, R, false><<<blocks, block, 0, st>>>(a);
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

// A thread makes one block of the generator, 8 values of 16 bits. 65,536 rows of 1,024 in bf16: with a residual 63 us, 98% of a plain copy's
// rate, without 55 (74%: there the generator's 20 wide products, 40 exclusive ors and 20 key sums for 8 values count). Loads asked
// for before the generator runs, or two blocks at a time, took longer (74 and 81 us).
template <class T, bool WIDE>
__global__ void __launch_bounds__(256, 8) k_dropout(const __grid_constant__ Drop a) {
    const uint64_t seed = (uint64_t)(a.seed ? *a.seed : a.seed_value);
    for (long long block = blockIdx.x * 256ll + threadIdx.x; block * 8 < a.n; block += gridDim.x * 256ll) {
        const uint4 r = philox(make_uint4((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)a.call, (uint32_t)(a.call >> 32)),
                               (uint32_t)seed, (uint32_t)(seed >> 32));
        // (a half is at least `least` where the word from it on is at least that, shifted up)
        const uint32_t bits[8] = {r.x << 16, r.x, r.y << 16, r.y, r.z << 16, r.z, r.w << 16, r.w}, least = a.least << 16;
        const T* x = reinterpret_cast<const T*>(a.x) + block * 8;
        const T* add = a.add ? reinterpret_cast<const T*>(a.add) + block * 8 : nullptr;
        T* y = reinterpret_cast<T*>(a.y) + block * 8;
        constexpr int V = 16 / (int)sizeof(T);
        if (WIDE && block * 8 + 8 <= a.n) {
#pragma unroll
            for (int u = 0; u < 8; u += V) {
                const Unit<T, V> v = load<T, V>(x + u);
                Unit<T, V> r{};
                float o[V];
                if (add) r = load<T, V>(add + u);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float b = add ? to_f(r.v[i]) : 0.f;
                    o[i] = bits[u + i] >= least ? fmaf(to_f(v.v[i]), a.by, b) : b;
                }
                store<T, V>(y + u, o);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (block * 8 + i >= a.n) break;
                const float o = add ? to_f(add[i]) : 0.f;
                y[i] = from_f<T>(bits[i] >= least ? fmaf(to_f(x[i]), a.by, o) : o);
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
