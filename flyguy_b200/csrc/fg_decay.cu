// Linear attention with a constant decay for each head, over whole recordings and for a single tick.
//
//   S_t = gamma S_{t-1} + k_t v_t^T,  o_t = scale q_t S_t,  gamma = exp(log_decay[h])          (forward)
//   R_t = gamma R_{t+1} + scale q_t go_t^T, R_last += gstate_out                              (backward, from the end)
//   gq_t = scale S_t go_t,  gk_t = R_t v_t,  gv_t = R_t^T k_t,  gstate = gamma R_0
//
// All four products are one scan with other operands, run from the front or from the back:
//   o  = scan(q, k, v)   gq = scan(go, v, k)   gv = scan'(k, q, go)   gk = scan'(v, go, q)
// The states of gq and gk are those of o and gv transposed.
//
// Few long recordings: the ticks of each are split into parts; a first launch leaves every part's own state (from
// zero) in the workspace, the second starts each part from the decayed sum of the states before it.
#include <type_traits>

#include "fg_memory.cuh"

namespace {
using namespace fgm;

constexpr int kMaxDim = 256;

struct Operand {
    char* p;
    long long batch, tick, head;
    int share;               // query heads to one head of this operand
};
// One scan: out_t = scale_out a_t S_t, S = gamma S + scale_in b c^T with a, b [.., D], c [.., E].
struct Scan {
    Operand a, b, c, out;
    int out_f32;             // out is fp32 (a partial result per query head)
    int beside;              // may run beside the launch before it: it reads nothing that one writes, and writes nothing that one touches
    const float* log_decay;
    const float* first;      // the state before the scan's first tick, or NULL
    float* last;             // the state after its last, or NULL
    int first_t, last_t;     // they lie [E][D] instead of [D][E]
    int backward;            // from the last tick to the first; first then counts undecayed at its tick, last decays once more
    const long long* offsets;
    long long batch, ticks;
    int heads, D, E, parts;
    float scale_in, scale_out;
    float* partial;          // [batch][heads][parts][D][E]: the parts' own states
};

struct Span {
    long long start, n;      // ticks of the recording
};
__device__ __forceinline__ Span span_of(const Scan& s, long long b) {
    if (!s.offsets) return {0, s.ticks};
    const long long lo = min(max(s.offsets[b], 0ll), s.ticks), hi = min(max(s.offsets[b + 1], lo), s.ticks);
    return {lo, hi - lo};
}
// gamma^n; n = 0 is 1 also for gamma = 0. Repeated multiplication goes by x + x (gamma - 1) instead: gamma close to 1 has
// no room for its last digits in fp32 (off by 1e-4 over the 3,000 ticks that it remembers), gamma - 1 has.
__device__ __forceinline__ float power(float log_decay, float n) { return n > 0.f ? expf(log_decay * n) : 1.f; }

// Scans that need nothing of one another overlap: a launch that may run beside the one before it begins once all of that
// one's blocks have begun, and takes the SMs that its last blocks leave free. 512 blocks on 148 SMs are 3.5 rounds: 64
// recordings of 1,024 ticks, 8 heads of 128 in bf16, forward and the three scans back take 650 us, in turn 719 (pass after
// pass; with the L2 flushed in between 707 and 755). What follows must follow both, so one block of the later launch ends after
// the earlier one has. (With parts the launch before is the parts', whose states are read.)
__device__ __forceinline__ void next_may_begin() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... Rest>
void launch_beside(void (*kernel)(Scan, Rest...), dim3 grid, int threads, int bytes, cudaStream_t st, Scan s, const Rest&... rest) {
    s.beside = s.beside && s.parts == 1;
    cudaLaunchAttribute beside{};
    beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    beside.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t how{};
    how.gridDim = grid;
    how.blockDim = dim3(threads);
    how.dynamicSmemBytes = bytes;
    how.stream = st;
    how.attrs = &beside;
    how.numAttrs = s.beside ? 1 : 0;
    MCK(cudaLaunchKernelEx(&how, kernel, s, rest...));
}

// ticks of a recording in one part: whole blocks of kAlign
constexpr int kAlign = 128;
__device__ __forceinline__ long long part_ticks(long long n, int parts) {
    const long long per = (n + parts - 1) / parts;
    return (per + kAlign - 1) / kAlign * kAlign;
}

}  // namespace
#include "fg_decay_mma.cuh"
#include "fg_decay_tc.cuh"
namespace {

// The recurrence itself, in fp32, for any type, size and stride: a block of 8 warps owns 32 columns of one head's
// state; lane = column, warp w holds rows w R .. w R + R - 1 in registers. 16 ticks of a and b are staged in shared
// memory as fp32 and read as broadcasts; the warps' shares of out meet in shared memory once per 16 ticks. It is what runs
// for a dim or value_dim over 128, where neither of the other kernels has room for the state. Bound by the multiply-adds,
// two a value of S and tick on the fp32 units, and the barriers between 16 ticks: 32 recordings of 509 ticks, 4 heads of 64 in
// fp32 with gradients take 2,825 us here and 379 as products of chunks (bf16, 64 of 1,024, 8 heads of 128: 49,100 and 720).
constexpr int kRecTicks = 16, kRecWarps = 8, kRecCols = 32;
constexpr int kRecRows = kMaxDim / kRecWarps;

template <class T>
__global__ void __launch_bounds__(32 * kRecWarps) k_decay_rec(const __grid_constant__ Scan s, int store_parts) {
    __shared__ __align__(16) float sa[kRecTicks][kMaxDim], sb[kRecTicks][kMaxDim];
    __shared__ float so[kRecTicks][kRecWarps][kRecCols];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int part = blockIdx.y;
    long long item = blockIdx.x;
    const int tiles = (s.E + kRecCols - 1) / kRecCols;
    const int tile = (int)(item % tiles);
    item /= tiles;
    const int h = (int)(item % s.heads);
    const long long b = item / s.heads;
    const Span sp = span_of(s, b);
    const long long per = part_ticks(sp.n, s.parts), t0 = min(sp.n, part * per), t1 = min(sp.n, t0 + per);
    const int R = (s.D + kRecWarps - 1) / kRecWarps, d0 = w * R;
    const int e = tile * kRecCols + lane;
    const bool col = e < s.E;
    const float ld = s.log_decay[h], fade = expm1f(ld);
    float S[kRecRows];
#pragma unroll
    for (int r = 0; r < kRecRows; ++r) S[r] = 0.f;

    // the state before this part
    const long long state0 = (b * s.heads + h) * s.D * s.E;
    if (!store_parts && (part == 0 || t1 > t0)) {
        if (s.first && col) {
            const float f = power(ld, (float)(s.backward ? max(t0 - 1, 0ll) : t0));
#pragma unroll
            for (int r = 0; r < kRecRows; ++r)
                if (r < R && d0 + r < s.D)
                    S[r] = f * s.first[state0 + (s.first_t ? (long long)e * s.D + d0 + r : (long long)(d0 + r) * s.E + e)];
        }
        for (int p = 0; p < part; ++p) {
            const float f = power(ld, (float)(t0 - min(sp.n, (p + 1) * per)));
            const float* q = s.partial + ((b * s.heads + h) * s.parts + p) * s.D * s.E;
#pragma unroll
            for (int r = 0; r < kRecRows; ++r)
                if (r < R && d0 + r < s.D && col) S[r] = fmaf(f, q[(long long)(d0 + r) * s.E + e], S[r]);
        }
    }
    bool undecayed = s.backward && s.first && part == 0 && !store_parts;   // the tick that `first` counts at fully

    auto row = [&](const Operand& o, long long t) {
        const long long tick = sp.start + (s.backward ? sp.n - 1 - t : t);
        return (s.offsets ? 0 : b * o.batch) + tick * o.tick + (h / o.share) * o.head;
    };
    for (long long t = t0; t < t1; t += kRecTicks) {
        const int n = (int)min((long long)kRecTicks, t1 - t);
        for (int i = threadIdx.x; i < n * s.D; i += 32 * kRecWarps) {
            const int j = i / s.D, d = i - j * s.D;
            sb[j][d] = to_f(reinterpret_cast<const T*>(s.b.p)[row(s.b, t + j) + d]) * s.scale_in;
            if (!store_parts) sa[j][d] = to_f(reinterpret_cast<const T*>(s.a.p)[row(s.a, t + j) + d]);
        }
        __syncthreads();
        for (int j = 0; j < n; ++j) {
            const float v = col ? to_f(reinterpret_cast<const T*>(s.c.p)[row(s.c, t + j) + e]) : 0.f;
            const float g = undecayed ? 0.f : fade;
            undecayed = false;
            float o = 0.f;
#pragma unroll
            for (int r = 0; r < kRecRows; ++r) {
                if (r < R && d0 + r < s.D) {
                    S[r] = fmaf(sb[j][d0 + r], v, fmaf(S[r], g, S[r]));
                    if (!store_parts) o = fmaf(sa[j][d0 + r], S[r], o);
                }
            }
            if (!store_parts) so[j][w][lane] = o;
        }
        __syncthreads();
        if (!store_parts)
            for (int j = w; j < n; j += kRecWarps) {
                float o = 0.f;
#pragma unroll
                for (int k = 0; k < kRecWarps; ++k) o += so[j][k][lane];
                if (col) {
                    const long long at = row(s.out, t + j) + e;
                    if (s.out_f32) reinterpret_cast<float*>(s.out.p)[at] = o * s.scale_out;
                    else reinterpret_cast<T*>(s.out.p)[at] = from_f<T>(o * s.scale_out);
                }
            }
        __syncthreads();
    }

    if (!col) return;
    if (store_parts) {
        float* q = s.partial + ((b * s.heads + h) * s.parts + part) * s.D * s.E;
#pragma unroll
        for (int r = 0; r < kRecRows; ++r)
            if (r < R && d0 + r < s.D) q[(long long)(d0 + r) * s.E + e] = S[r];
        return;
    }
    // the part with the last tick (the first part of a recording without ticks) hands the state on
    if (s.last && (sp.n ? t1 == sp.n && t1 > t0 : part == 0)) {
        const float f = s.backward && sp.n ? power(ld, 1.f) : 1.f;
#pragma unroll
        for (int r = 0; r < kRecRows; ++r)
            if (r < R && d0 + r < s.D)
                s.last[state0 + (s.last_t ? (long long)e * s.D + d0 + r : (long long)(d0 + r) * s.E + e)] = f * S[r];
    }
}

// out[tick][key head][:] = the fp32 results of the query heads that share it, added in order; V values a thread. Bound by
// the memory: 97,500 ticks, 8 heads of 64 to 2 take 35 us, 6.1 TB/s (a value a thread with 64-bit divisions: 99 us).
template <class T, int V, class Index>
__global__ void __launch_bounds__(256) k_share_sum(const float* __restrict__ in, Operand out, Index ticks, int heads,
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
void share_sum(const float* in, const Operand& out, long long batch, long long ticks, int heads, int key_heads, int dim, cudaStream_t st) {
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
void clear_outside(const fg_decay_args* g, const fg_ticks* const (&to)[3], const long long (&heads)[3], const long long (&dims)[3], int n, int size,
                   cudaStream_t st) {
    if (!g->offsets || !g->ticks) return;
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
        most = std::max(most, g->ticks * heads[i] * (dims[i] / values));
    }
    a.offsets = g->offsets;
    a.batch = g->batch;
    a.ticks = g->ticks;
    auto* kernel = piece == 16 ? k_clear_outside<uint4> : piece == 4 ? k_clear_outside<uint32_t> : k_clear_outside<uint16_t>;
    kernel<<<dim3((unsigned)std::min<long long>((most + 255) / 256, kSms), n), 256, 0, st>>>(a);
    MCK(cudaGetLastError());
}

// A single tick: a block per (row, head). A warp takes every 8th row of the state, its lanes the columns; state in and
// out are the whole cost. For value_dims that are no multiple of 4 (2,048 rows, 8 heads of 128 x 128: 744 us, below 333).
template <class T>
__global__ void __launch_bounds__(256) k_decay_step(Operand q, Operand k, Operand v, Operand out,
                                                    const float* __restrict__ log_decay, float* __restrict__ state,
                                                    const long long* __restrict__ slots, long long n_slots, int heads,
                                                    int D, int E, float scale) {
    __shared__ float so[8][kMaxDim];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long b = blockIdx.x / heads;
    const int h = (int)(blockIdx.x - b * heads);
    const long long slot = slots ? slots[b] : b;
    T* o = reinterpret_cast<T*>(out.p) + b * out.batch + h * out.head;
    if (slot < 0 || slot >= n_slots) {
        for (int e = threadIdx.x; e < E; e += 256) o[e] = from_f<T>(0.f);
        return;
    }
    const T* qp = reinterpret_cast<const T*>(q.p) + b * q.batch + h * q.head;
    const T* kp = reinterpret_cast<const T*>(k.p) + b * k.batch + (h / k.share) * k.head;
    const T* vp = reinterpret_cast<const T*>(v.p) + b * v.batch + (h / v.share) * v.head;
    float* S = state + (slot * heads + h) * D * E;
    const float fade = expm1f(log_decay[h]);
    for (int e = lane; e < E; e += 32) {
        const float ve = to_f(vp[e]);
        float acc = 0.f;
        for (int d = w; d < D; d += 8) {
            const float old = S[(long long)d * E + e];
            const float x = fmaf(to_f(kp[d]), ve, fmaf(old, fade, old));
            S[(long long)d * E + e] = x;
            acc = fmaf(to_f(qp[d]), x, acc);
        }
        so[w][e] = acc;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 256) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += so[i][e];
        o[e] = from_f<T>(s * scale);
    }
}

// The same with value_dim a multiple of 4 and 16-byte aligned: a thread owns 4 columns of every R-th row, and asks for 8 rows
// before it uses the first: state in and out is all there is to a tick, 16 bytes a load. 2,048 rows, 8 heads of 128 x 128:
// 333 us, 6.5 TB/s, 99% of a plain copy's rate. One tick of 8 rows is one wait for the memory; the call costs 14 us, most of
// it on the host.
template <class T>
__global__ void __launch_bounds__(256, 3) k_decay_step4(Operand q, Operand k, Operand v, Operand out,
                                                        const float* __restrict__ log_decay, float* __restrict__ state,
                                                        const long long* __restrict__ slots, long long n_slots, int heads,
                                                        int D, int E, float scale) {
    __shared__ float sq[kMaxDim], sk[kMaxDim];
    __shared__ float4 so[256];
    const int h = blockIdx.x % heads;
    const long long b = blockIdx.x / heads;
    const long long slot = slots ? slots[b] : b;
    T* o = reinterpret_cast<T*>(out.p) + b * out.batch + h * out.head;
    if (slot < 0 || slot >= n_slots) {
        for (int e = threadIdx.x; e < E; e += 256) o[e] = from_f<T>(0.f);
        return;
    }
    const int C = E / 4, R = 256 / C, r = threadIdx.x / C, c = threadIdx.x - r * C;
    const bool busy = r < R;
    float4* S = reinterpret_cast<float4*>(state + (slot * heads + h) * D * E) + c;
    constexpr int kAhead = 8;
    float4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (busy && r + i * R < D) x[i] = S[(r + i * R) * C];
    const T* qp = reinterpret_cast<const T*>(q.p) + b * q.batch + h * q.head;
    const T* kp = reinterpret_cast<const T*>(k.p) + b * k.batch + (h / k.share) * k.head;
    const T* vp = reinterpret_cast<const T*>(v.p) + b * v.batch + (h / v.share) * v.head;
    for (int d = threadIdx.x; d < D; d += 256) {
        sq[d] = to_f(qp[d]);
        sk[d] = to_f(kp[d]);
    }
    float ve[4] = {0.f, 0.f, 0.f, 0.f};
    if (busy) {
#pragma unroll
        for (int i = 0; i < 4; ++i) ve[i] = to_f(vp[4 * c + i]);
    }
    const float fade = expm1f(log_decay[h]);
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int d0 = r; busy && d0 < D; d0 += kAhead * R) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int d = d0 + i * R;
            if (d >= D) break;
            float4 s = x[i];
            const float kd = sk[d], qd = sq[d];
            s.x = fmaf(kd, ve[0], fmaf(s.x, fade, s.x));
            s.y = fmaf(kd, ve[1], fmaf(s.y, fade, s.y));
            s.z = fmaf(kd, ve[2], fmaf(s.z, fade, s.z));
            s.w = fmaf(kd, ve[3], fmaf(s.w, fade, s.w));
            S[d * C] = s;
            acc.x = fmaf(qd, s.x, acc.x);
            acc.y = fmaf(qd, s.y, acc.y);
            acc.z = fmaf(qd, s.z, acc.z);
            acc.w = fmaf(qd, s.w, acc.w);
            if (d + kAhead * R < D) x[i] = S[(d + kAhead * R) * C];
        }
    }
    so[threadIdx.x] = acc;
    __syncthreads();
    const float* sums = reinterpret_cast<const float*>(so);
    for (int e = threadIdx.x; e < E; e += 256) {
        float s = 0.f;
        for (int i = 0; i < R; ++i) s += sums[i * E + e];
        o[e] = from_f<T>(s * scale);
    }
}

Operand operand(const fg_ticks& t, long long share) {
    return {static_cast<char*>(t.p), t.batch, t.tick, t.head, (int)share};
}

struct Sizes {
    long long batch, ticks, heads, key_heads, D, E;
};
void check_sizes(const Sizes& z, const char* who) {
    const std::string w = who;
    if (z.batch < 0 || z.ticks < 0) throw MemErr{w + ": a negative size"};
    if (z.heads < 1 || z.key_heads < 1 || z.heads % z.key_heads || z.heads > 65535)
        throw MemErr{w + ": heads must be a multiple of key_heads, 1 to 65535"};
    if (z.D < 1 || z.D > kMaxDim || z.E < 1 || z.E > kMaxDim) throw MemErr{w + ": dim and value_dim must be 1 to 256"};
    if (z.batch * z.heads > (1ll << 27)) throw MemErr{w + ": batch * heads is over 2^27"};
}

// Parts a recording. A part costs its b and c read twice, so: as many as keep the blocks within one round of the SMs (the
// tcgen05 kernel takes a SM to itself, two blocks of the mma.sync kernel share one), of at least four chunks. The
// recurrence's blocks are slow and share a SM: more of them. (1 recording of 65,536 ticks, 8 heads of 128 in bf16: 289 us in 18
// parts a head; unsplit, 512 chunks of 4.7 us follow one another.)
int parts_of(const fg_decay_args* g) {
    const long long rows = std::max<long long>(1, g->batch * g->heads);
    const long long mean = g->offsets ? g->ticks / std::max<long long>(1, g->batch) : g->ticks;
    const bool mma = g->dim <= 128 && g->value_dim <= 128;
    const bool tc = mma && g->type == FG_BF16 && g->dim % 16 == 0 && g->value_dim % 16 == 0;
    const long long blocks = mma ? rows : rows * ((std::min(g->dim, g->value_dim) + kRecCols - 1) / kRecCols);
    const long long want = (tc ? kSms : mma ? 2 * kSms : 4 * kSms) / blocks, most = mean / (tc ? 512 : 256);
    return (int)std::min<long long>(64, std::max<long long>(1, std::min(want, most)));
}
long long partial_floats(const fg_decay_args* g) {
    const int parts = parts_of(g);
    return parts > 1 ? g->batch * g->heads * parts * g->dim * g->value_dim : 0;
}
long long all_ticks(const fg_decay_args* g) { return g->offsets ? g->ticks : g->batch * g->ticks; }
long long work_floats(const fg_decay_args* g, bool backward) {
    const auto whole = [](long long n) { return (n + 3) / 4 * 4; };   // (each part begins at 16 bytes)
    long long n = whole(partial_floats(g));
    if (backward && g->heads != g->key_heads) n += whole(all_ticks(g) * g->heads * g->dim) + whole(all_ticks(g) * g->heads * g->value_dim);
    return n;
}

void check(const fg_decay_args* g, bool backward) {
    const char* who = backward ? "fg_decay_attn_bwd" : "fg_decay_attn";
    need(g, "fg_decay_attn: no arguments");
    check_sizes({g->batch, g->ticks, g->heads, g->key_heads, g->dim, g->value_dim}, who);
    need(g->type >= FG_F32 && g->type <= FG_F16, "fg_decay_attn: unknown type");
    need(g->log_decay, "fg_decay_attn: log_decay is NULL");
    const bool used = g->batch && g->ticks;
    need(!used || (g->q.p && g->k.p && g->v.p && (backward ? g->go.p && g->gq.p && g->gk.p && g->gv.p : g->o.p != nullptr)),
         "fg_decay_attn: null pointer");
    need(backward || !g->state || g->state != g->state_out, "fg_decay_attn: state and state_out are the same");
    need(!backward || !g->gstate || (g->gstate != g->state && g->gstate != g->gstate_out),
         "fg_decay_attn_bwd: gstate is state or gstate_out");
    const long long bytes = work_floats(g, backward) * 4;
    need(!bytes || (g->work && g->work_bytes >= bytes), "fg_decay_attn: the workspace is too small");
    need(reinterpret_cast<uintptr_t>(g->work) % 16 == 0, "fg_decay_attn: the workspace is not 16-byte aligned");
}

Scan scan_of(const fg_decay_args* g) {
    Scan s{};
    s.log_decay = g->log_decay;
    s.offsets = g->offsets;
    s.batch = g->batch;
    s.ticks = g->ticks;
    s.heads = (int)g->heads;
    s.D = (int)g->dim;
    s.E = (int)g->value_dim;
    s.parts = parts_of(g);
    s.scale_in = 1.f;
    s.scale_out = (float)g->scale;
    s.partial = static_cast<float*>(g->work);
    return s;
}

// By what fits: bf16 tiles that TMA takes go to the tcgen05 kernel, other types and strides up to 128 to mma.sync (fp32
// needs its terms; 64 recordings of 1,024 ticks, 8 heads of 128 with gradients: 720 us and, in fp16, 5.4 ms), the rest to the recurrence.
template <class T>
void launch(const Scan& s, cudaStream_t st) {
    if (std::is_same<T, __nv_bfloat16>::value && tc_fits(s)) return tc_launch(s, st);
    if (s.D <= 128 && s.E <= 128) return s.backward ? mma_launch_dims<T, true>(s, st) : mma_launch_dims<T, false>(s, st);
    const long long blocks = s.batch * s.heads * ((s.E + kRecCols - 1) / kRecCols);
    if (s.parts > 1) k_decay_rec<T><<<dim3((unsigned)blocks, s.parts - 1), 32 * kRecWarps, 0, st>>>(s, 1);
    k_decay_rec<T><<<dim3((unsigned)blocks, s.parts), 32 * kRecWarps, 0, st>>>(s, 0);
    MCK(cudaGetLastError());
}

}  // namespace

extern "C" {

int fg_decay_attn(const fg_decay_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, false);
        clear_outside(g, {&g->o}, {g->heads}, {g->value_dim}, 1, g->type == FG_F32 ? 4 : 2, static_cast<cudaStream_t>(stream));
        if (!g->batch) return 0;
        const long long share = g->heads / g->key_heads;
        Scan s = scan_of(g);
        s.a = operand(g->q, 1);
        s.b = operand(g->k, share);
        s.c = operand(g->v, share);
        s.out = operand(g->o, 1);
        s.first = g->state;
        s.last = g->state_out;
        by_type(g->type, [&](auto t) { launch<decltype(t)>(s, static_cast<cudaStream_t>(stream)); });
        return 0;
    });
}

int fg_decay_attn_bwd(const fg_decay_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, true);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const auto clear = [&] {                              // (last: sums of shared heads go over all ticks)
            clear_outside(g, {&g->gq, &g->gk, &g->gv}, {g->heads, g->key_heads, g->key_heads}, {g->dim, g->dim, g->value_dim}, 3,
                          g->type == FG_F32 ? 4 : 2, st);
        };
        if (!g->batch) {
            clear();
            return 0;
        }
        const long long share = g->heads / g->key_heads;
        float* for_gv = static_cast<float*>(g->work) + (partial_floats(g) + 3) / 4 * 4;
        float* for_gk = for_gv + (all_ticks(g) * g->heads * g->value_dim + 3) / 4 * 4;
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            Scan s = scan_of(g);
            std::swap(s.D, s.E);                              // gq = scan(go, v, k), its states transposed
            s.a = operand(g->go, 1);
            s.b = operand(g->v, share);
            s.c = operand(g->k, share);
            s.out = operand(g->gq, 1);
            s.first = g->state;
            s.first_t = 1;
            launch<T>(s, st);
            // the gradients of shared heads: per query head in fp32, then added
            auto shared = [&](Scan x, const fg_ticks& to, long long dim, float* wide) {
                x.out = share > 1 ? Operand{reinterpret_cast<char*>(wide), g->ticks * g->heads * dim, g->heads * dim, dim, 1} : operand(to, 1);
                x.out_f32 = share > 1;
                x.beside = 1;
                launch<T>(x, st);
            };
            auto add = [&](const fg_ticks& to, long long dim, const float* wide) {
                if (share > 1 && all_ticks(g))
                    share_sum<T>(wide, operand(to, 1), g->offsets ? 1 : g->batch, g->ticks, (int)g->heads, (int)g->key_heads, (int)dim, st);
            };
            s = scan_of(g);                                   // gv = scan'(k, q, go)
            s.backward = 1;
            std::swap(s.scale_in, s.scale_out);
            s.a = operand(g->k, share);
            s.b = operand(g->q, 1);
            s.c = operand(g->go, 1);
            s.first = g->gstate_out;
            s.last = g->gstate;
            shared(s, g->gv, g->value_dim, for_gv);
            std::swap(s.D, s.E);                              // gk = scan'(v, go, q), its states transposed
            s.a = operand(g->v, share);
            std::swap(s.b, s.c);
            s.first_t = 1;
            s.last = nullptr;
            shared(s, g->gk, g->dim, for_gk);
            add(g->gv, g->value_dim, for_gv);
            add(g->gk, g->dim, for_gk);
        });
        clear();
        return 0;
    });
}

long long fg_decay_work(const fg_decay_args* g, int backward) {
    return mem_guard([&]() -> long long {
        need(g, "fg_decay_attn: no arguments");
        check_sizes({g->batch, g->ticks, g->heads, g->key_heads, g->dim, g->value_dim}, "fg_decay_work");
        return work_floats(g, backward != 0) * 4;
    });
}

int fg_decay_step(const fg_step_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        need(g, "fg_decay_step: no arguments");
        check_sizes({g->batch, 1, g->heads, g->key_heads, g->dim, g->value_dim}, "fg_decay_step");
        need(g->n_slots >= 0, "fg_decay_step: a negative size");
        need(g->log_decay, "fg_decay_step: log_decay is NULL");
        if (!g->batch) return 0;
        need(g->q.p && g->k.p && g->v.p && g->o.p && (g->state || !g->n_slots), "fg_decay_step: null pointer");
        const long long share = g->heads / g->key_heads;
        const bool by4 = g->value_dim % 4 == 0 && reinterpret_cast<uintptr_t>(g->state) % 16 == 0;
        by_type(g->type, [&](auto t) {
            auto* kernel = by4 ? k_decay_step4<decltype(t)> : k_decay_step<decltype(t)>;
            kernel<<<(unsigned)(g->batch * g->heads), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                operand(g->q, 1), operand(g->k, share), operand(g->v, share), operand(g->o, 1), g->log_decay, g->state,
                g->slots, g->n_slots, (int)g->heads, (int)g->dim, (int)g->value_dim, (float)g->scale);
        });
        MCK(cudaGetLastError());
        return 0;
    });
}

int fg_mem_sync(void* stream) {
    return (int)mem_guard([&]() -> long long {
        int bad = 0;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        MCK(cudaMemcpyFromSymbolAsync(&bad, g_tc_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
        MCK(cudaStreamSynchronize(st));
        need(!bad, "fg_decay_attn: a wait on the tensor cores ran out; its results are not to be used");
        return 0;
    });
}

const char* fg_mem_last_error(void) { return last_error().c_str(); }

}  // extern "C"

namespace fgm {
std::string& last_error() {
    static thread_local std::string e;
    return e;
}
}  // namespace fgm
