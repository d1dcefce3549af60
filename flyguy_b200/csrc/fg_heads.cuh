// What the attentions with a state share around their kernels: gradients of heads that several others read, and ticks that no recording covers.
#pragma once
#include <type_traits>

#include "fg_memory.cuh"

namespace {
using namespace fgm;

// out[tick][key head][:] = the fp32 results of the query heads that share it, added in order; V values a thread. Bound by
// the memory: 97,500 ticks, 8 heads of 64 to 2 take 35 us, 6.1 TB/s (a value a thread with 64-bit divisions: 99 us).
template <class T, int V, class Index>
__global__ void __launch_bounds__(256) k_share_sum(const float* __restrict__ in, fg_ticks out, Index ticks, int heads,
                                                   int key_heads, int dim, Index units) {
    const int share = heads / key_heads, of_row = dim / V;
    using Load = std::conditional_t<V == 4, float4, float>;
    for (Index i = blockIdx.x * (Index)blockDim.x + threadIdx.x; i < units; i += gridDim.x * (Index)blockDim.x) {
        const Index row = i / of_row;
        const int d = (int)(i - row * of_row) * V;
        const Index tick = row / key_heads, b = tick / ticks;
        const int h = (int)(row - tick * key_heads);
        const float* p = in + ((long long)tick * heads + h * share) * dim + d;
        float s[V] = {};
#pragma unroll 4
        for (int k = 0; k < share; ++k) {
            const Load v = *reinterpret_cast<const Load*>(p + (long long)k * dim);
            const float* x = reinterpret_cast<const float*>(&v);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += x[j];
        }
        T* to = reinterpret_cast<T*>(out.p) + (long long)b * out.batch + (long long)(tick - b * ticks) * out.tick + h * out.head + d;
#pragma unroll
        for (int j = 0; j < V; ++j) to[j] = from_f<T>(s[j]);
    }
}
template <class T>
void share_sum(const float* in, const fg_ticks& out, long long batch, long long ticks, int heads, int key_heads, int dim, cudaStream_t st) {
    const bool four = dim % 4 == 0;                          // (`in` is the workspace's: aligned)
    const long long units = batch * ticks * key_heads * dim / (four ? 4 : 1);
    const unsigned blocks = (unsigned)std::min<long long>((units + 255) / 256, kSms * 32);
    const bool small = units < (1ll << 31) - kSms * 32 * 256;  // 32-bit divisions: a third of the time
    if (small && four) k_share_sum<T, 4, uint32_t><<<blocks, 256, 0, st>>>(in, out, (uint32_t)ticks, heads, key_heads, dim, (uint32_t)units);
    else if (small) k_share_sum<T, 1, uint32_t><<<blocks, 256, 0, st>>>(in, out, (uint32_t)ticks, heads, key_heads, dim, (uint32_t)units);
    else k_share_sum<T, 1, long long><<<blocks, 256, 0, st>>>(in, out, ticks, heads, key_heads, dim, batch * ticks * key_heads * dim);
    MCK(cudaGetLastError());
}

// Zeros for the ticks that no recording covers, before the first and after the last (a packed buffer with room to spare): the
// scans write recordings only, and what reads these outputs, the gradient of a projection's weights say, sums over all ticks.
// Rows of `units` pieces of U of each head; up to three outputs, one a grid row. With nothing to clear it is the cost of a launch,
// 3 us beside the scans' 190.
struct Outside {
    struct {
        char* p;
        long long tick, head;        // strides in pieces
        int heads, units;
    } out[3];
    const long long* offsets;
    long long batch, ticks;
};
template <class U>
__global__ void __launch_bounds__(256) k_clear_outside(const __grid_constant__ Outside a) {
    const auto& o = a.out[blockIdx.y];
    const long long lo = min(max(a.offsets[0], 0ll), a.ticks), hi = min(max(a.offsets[a.batch], lo), a.ticks);
    const long long row = (long long)o.heads * o.units, n = (lo + a.ticks - hi) * row;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long t = i / row;
        const int r = (int)(i - t * row), h = r / o.units;
        reinterpret_cast<U*>(o.p)[(t < lo ? t : hi + t - lo) * o.tick + h * o.head + r - h * o.units] = U{};
    }
}
// `n` outputs of heads[i] x dims[i] values of `size` bytes
inline void clear_outside(const long long* offsets, long long batch, long long ticks, const fg_ticks* const (&to)[3], const long long (&heads)[3],
                          const long long (&dims)[3], int n, int size, cudaStream_t st) {
    if (!offsets || !ticks) return;
    bool wide = true;                                        // pieces of 16 bytes
    for (int i = 0; i < n; ++i) {
        if (!to[i]->p) return;                               // (no recordings, and no outputs)
        wide = wide && reinterpret_cast<uintptr_t>(to[i]->p) % 16 == 0 && to[i]->tick * size % 16 == 0 && to[i]->head * size % 16 == 0 &&
               dims[i] * size % 16 == 0;
    }
    const int piece = wide ? 16 : size, values = piece / size;
    Outside a{};
    long long most = 1;
    for (int i = 0; i < n; ++i) {
        a.out[i] = {static_cast<char*>(to[i]->p), to[i]->tick / values, to[i]->head / values, (int)heads[i], (int)(dims[i] / values)};
        most = std::max(most, ticks * heads[i] * (dims[i] / values));
    }
    a.offsets = offsets;
    a.batch = batch;
    a.ticks = ticks;
    auto* kernel = piece == 16 ? k_clear_outside<uint4> : piece == 4 ? k_clear_outside<uint32_t> : k_clear_outside<uint16_t>;
    kernel<<<dim3((unsigned)std::min<long long>((most + 255) / 256, kSms), n), 256, 0, st>>>(a);
    MCK(cudaGetLastError());
}

}  // namespace
