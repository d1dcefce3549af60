// The gated delta rule: a linear attention whose state forgets by a gate of each tick and overwrites what a key held before.
//
//   S_t = g_t S_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - g_t k_t S_{t-1}),  o_t = scale q_t S_t,  g_t = exp(log_decay_t)
//
// Over recordings by chunks (fg_delta_chain.cuh), with the gradients of all inputs (fg_delta_grad.cuh), and for a single tick below.
#include <type_traits>

#include "fg_delta_grad.cuh"

namespace {

constexpr int kMaxDim = 128, kMaxValue = 256, kMaxStep = 256;

// ---- a single tick ------------------------------------------------------------------------------------------------------

struct Step {
    fg_ticks q, k, v, o;
    const float *log_decay, *beta;
    long long log_batch, log_head, beta_batch, beta_head;
    float* state;
    const long long* slots;
    long long n_slots;
    int heads, q_share, k_share, v_share, D, E, tiles;
    float scale;
};
// A block takes 32 columns of a row's state of one head, whole in registers: V columns a thread of every (256 V / 32)-th row. One
// pass over them gives k S and q S, and o = q S + (q k) u needs no second one: PER values a column. State in and out is the cost.
template <class T, int V, int PER>
__global__ void __launch_bounds__(256, PER * V <= 16 ? 5 : 3) k_delta_step(const __grid_constant__ Step s) {
    constexpr int kAcross = 32 / V, kRows = 256 / kAcross, kPer = PER;
    __shared__ float sq[kMaxStep], sk[kMaxStep], pred[8][32], out[8][32], qk_part[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long item = blockIdx.x;
    const int tile = (int)(item % s.tiles);
    item /= s.tiles;
    const int h = (int)(item % s.heads), r = tid / kAcross, c = tid % kAcross, e0 = tile * 32 + c * V;
    const long long b = item / s.heads, slot = s.slots ? s.slots[b] : b;
    T* o = reinterpret_cast<T*>(s.o.p) + b * s.o.batch + h * s.o.head;
    if (slot < 0 || slot >= s.n_slots) {
        if (tid < 32 && tile * 32 + tid < s.E) o[tile * 32 + tid] = from_f<T>(0.f);
        return;
    }
    float* S = s.state + (slot * s.heads + h) * s.D * s.E + e0;
    const bool in = e0 < s.E;
    float x[kPer][V];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = r + i * kRows;
        if (in && d < s.D) {
            if constexpr (V == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(S + (long long)d * s.E);
            else x[i][0] = S[(long long)d * s.E];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = 0.f;
        }
    }
    const T* qp = reinterpret_cast<const T*>(s.q.p) + b * s.q.batch + (h / s.q_share) * s.q.head;
    const T* kp = reinterpret_cast<const T*>(s.k.p) + b * s.k.batch + (h / s.k_share) * s.k.head;
    const T* vp = reinterpret_cast<const T*>(s.v.p) + b * s.v.batch + (h / s.v_share) * s.v.head;
    float qk = 0.f;
    {
        const float q = tid < s.D ? to_f(qp[tid]) : 0.f, k = tid < s.D ? to_f(kp[tid]) : 0.f;
        sq[tid] = q;
        sk[tid] = k;
        qk = warp_sum(q * k);
        if (lane == 0) qk_part[warp] = qk;
    }
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = in ? to_f(vp[e0 + j]) : 0.f;
    const float decay = expf(s.log_decay[b * s.log_batch + h * s.log_head]), beta = s.beta[b * s.beta_batch + h * s.beta_head];
    __syncthreads();
    float ks[V] = {}, qs[V] = {};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = r + i * kRows;
        if (d >= s.D) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            x[i][j] *= decay;
            ks[j] = fmaf(sk[d], x[i][j], ks[j]);
            qs[j] = fmaf(sq[d], x[i][j], qs[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int w = kAcross; w < 32; w <<= 1) {
            ks[j] += __shfl_xor_sync(0xffffffffu, ks[j], w);
            qs[j] += __shfl_xor_sync(0xffffffffu, qs[j], w);
        }
        if (lane < kAcross) {
            pred[warp][lane * V + j] = ks[j];
            out[warp][lane * V + j] = qs[j];
        }
    }
    __syncthreads();
    float u[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float p = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) p += pred[w][c * V + j];
        u[j] = beta * (v[j] - p);
    }
    if (in) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int d = r + i * kRows;
            if (d >= s.D) break;
#pragma unroll
            for (int j = 0; j < V; ++j) x[i][j] = fmaf(sk[d], u[j], x[i][j]);
            if constexpr (V == 4) *reinterpret_cast<float4*>(S + (long long)d * s.E) = *reinterpret_cast<const float4*>(x[i]);
            else S[(long long)d * s.E] = x[i][0];
        }
        if (r == 0) {
            qk = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) qk += qk_part[w];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float p = 0.f;
#pragma unroll
                for (int w = 0; w < 8; ++w) p += out[w][c * V + j];
                o[e0 + j] = from_f<T>(fmaf(qk, u[j], p) * s.scale);
            }
        }
    }
}

// Many rows: a block goes from one (row, head) to the next with three places for a state in shared memory. A warp of its own brings whole
// states as bulk copies, the next two while one is worked on, and sends them off again; 16 warps work, V = 4 columns a thread of every R-th
// row. D E at most 16,384 (64 KB), at most 32 values a thread.
constexpr int kWideThreads = 512, kWidePer = 8, kWidePlaces = 3, kWideSums = 2 * 16 * kWideThreads;
__device__ int g_step_error;              // a wait ran out (fg_mem_sync)
struct WideLayout {
    int state, bytes;                // of a place, of the block
    __host__ __device__ WideLayout(int D, int E) : state(D * E * 4), bytes(kWidePlaces * D * E * 4 + kWideSums + 4 * 5 * kMaxStep + 64) {}
};
// a phase of a barrier, given up after about 2 s (or so many times that)
__device__ __forceinline__ bool phase_of(uint32_t bar, uint32_t parity, int times = 1) {
    uint32_t done = 0;
    for (int tries = 0; !done && tries < 20000 * times; ++tries)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 100000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
    return done != 0;
}
// the workers' barrier; whether all of them say yes
__device__ __forceinline__ bool workers(bool yes) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.and.pred p, 1, 512, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)yes)
        : "memory");
    return all != 0;
}
template <class T>
__global__ void __launch_bounds__(kWideThreads + 32, 1) k_delta_step_wide(const __grid_constant__ Step s, uint32_t items) {
    static_assert(kWideThreads == 512, "the workers' barrier");
    extern __shared__ __align__(128) unsigned char smem[];
    const WideLayout lay(s.D, s.E);
    float4* part = reinterpret_cast<float4*>(smem + kWidePlaces * lay.state);          // [R][E / 4] of k S, then of q S
    float* row = reinterpret_cast<float*>(smem + kWidePlaces * lay.state + kWideSums);   // two places: k, q; then u
    uint64_t* bars = reinterpret_cast<uint64_t*>(row + 5 * kMaxStep);
    const int tid = threadIdx.x, C = s.E / 4, R = kWideThreads / C, r = tid / C, c = tid - r * C;
    const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem), full = (uint32_t)__cvta_generic_to_shared(bars), done = full + 8 * kWidePlaces;
    if (tid < 2 * kWidePlaces)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full + 8 * tid), "r"(tid < kWidePlaces ? 1 : kWideThreads / 32) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    // this block's i-th item is blockIdx.x + i gridDim.x; its state goes to place i mod 3. An item without a slot uses no place.
    const auto nth = [&](uint32_t i) { return blockIdx.x + i * gridDim.x; };
    const auto slot_of = [&](uint32_t item) {
        const uint32_t b = item / (uint32_t)s.heads;
        const long long slot = s.slots ? s.slots[b] : b;
        return slot >= 0 && slot < s.n_slots ? slot : -1;
    };
    if (tid >= kWideThreads) {
        if (tid != kWideThreads) return;
        uint32_t fetched = 0, phases = 0, open = 0;          // open: places whose copy has been asked for, and not answered by the workers
        long long slots[kWidePlaces];
        const auto fetch = [&]() {
            const uint32_t item = nth(fetched), place = fetched % kWidePlaces;
            ++fetched;
            if (item >= items) return;
            const long long slot = slots[place] = slot_of(item);
            if (slot < 0) return;
            open |= 1u << place;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8 * place), "r"(lay.state) : "memory");
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(sm + place * lay.state),
                         "l"(s.state + (slot * s.heads + item % (uint32_t)s.heads) * s.D * s.E), "r"(lay.state), "r"(full + 8 * place)
                         : "memory");
        };
        for (int i = 0; i < kWidePlaces; ++i) fetch();
        for (uint32_t i = 0; nth(i) < items; ++i) {
            const uint32_t place = i % kWidePlaces;
            if (slots[place] >= 0) {
                // (longer than the workers wait for this state: whatever they worked on is sent off)
                if (!phase_of(done + 8 * place, (phases >> place) & 1, 2)) {
                    atomicExch(&g_step_error, 1);
                    break;
                }
                phases ^= 1u << place;
                open &= ~(1u << place);
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                                 s.state + (slots[place] * s.heads + nth(i) % (uint32_t)s.heads) * s.D * s.E),
                             "r"(sm + place * lay.state), "r"(lay.state)
                             : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
            fetch();
        }
        // (after a wait that ran out) copies land before the block ends
        for (uint32_t place = 0; place < kWidePlaces; ++place)
            if (open >> place & 1) phase_of(full + 8 * place, (phases >> place) & 1);
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        return;
    }
    const bool busy = r < R;
    // what else an item needs, one item ahead in registers, as it comes (whatever is done to it here would wait for it)
    T nk = from_f<T>(0.f), nq = nk, nv = nk;
    float ndecay = 0.f, nbeta = 0.f;
    long long nslot = -1;
    const auto ahead = [&](uint32_t i) {
        const uint32_t item = nth(i);
        if (item >= items) return;
        const long long b = item / (uint32_t)s.heads;
        const int h = (int)(item - (uint32_t)b * (uint32_t)s.heads);
        nslot = s.slots ? s.slots[b] : b;
        if (tid < s.D) {
            nk = reinterpret_cast<const T*>(s.k.p)[b * s.k.batch + (h / s.k_share) * s.k.head + tid];
            nq = reinterpret_cast<const T*>(s.q.p)[b * s.q.batch + (h / s.q_share) * s.q.head + tid];
        }
        if (tid < s.E) nv = reinterpret_cast<const T*>(s.v.p)[b * s.v.batch + (h / s.v_share) * s.v.head + tid];
        ndecay = s.log_decay[b * s.log_batch + h * s.log_head];
        nbeta = s.beta[b * s.beta_batch + h * s.beta_head];
    };
    const auto out_of = [&](uint32_t item) {
        return reinterpret_cast<T*>(s.o.p) + (long long)(item / (uint32_t)s.heads) * s.o.batch + item % (uint32_t)s.heads * s.o.head;
    };
    ahead(0);
    uint32_t phases = 0;
    for (uint32_t i = 0; nth(i) < items; ++i) {
        const uint32_t place = i % kWidePlaces;
        const long long slot = nslot;
        float *sk = row + (i & 1) * 2 * kMaxStep, *sq = sk + kMaxStep;
        if (tid < s.D) {
            sk[tid] = to_f(nk);
            sq[tid] = to_f(nq);
        }
        const float v = to_f(nv), decay = expf(ndecay), beta = nbeta;
        ahead(i + 1);
        T* o = out_of(nth(i));
        workers(true);                                        // k and q are there
        if (slot < 0 || slot >= s.n_slots) {                  // (the same for all threads)
            for (int e = tid; e < s.E; e += kWideThreads) o[e] = from_f<T>(0.f);
            continue;
        }
        const bool there = phase_of(full + 8 * place, (phases >> place) & 1);
        phases ^= 1u << place;
        float4* S = reinterpret_cast<float4*>(smem + place * lay.state) + c;
        float4 x[kWidePer];
        float ks[4] = {}, qs[4] = {};
        if (busy) {
#pragma unroll
            for (int n = 0; n < kWidePer; ++n) {
                const int d = r + n * R;
                if (d >= s.D) break;
                x[n] = S[d * C];
                float* p = &x[n].x;
                const float kd = sk[d], qd = sq[d];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[j] *= decay;
                    ks[j] = fmaf(kd, p[j], ks[j]);
                    qs[j] = fmaf(qd, p[j], qs[j]);
                }
            }
            part[tid] = make_float4(ks[0], ks[1], ks[2], ks[3]);
            part[kWideThreads + tid] = make_float4(qs[0], qs[1], qs[2], qs[3]);
        }
        float qk = 0.f;
        for (int d = tid & 31; d < s.D; d += 32) qk = fmaf(sk[d], sq[d], qk);
        qk = warp_sum(qk);
        if (!workers(there)) {                                // (for all threads, if for one: this state and the block's later ones stay as they were)
            for (uint32_t k = i; nth(k) < items; ++k)
                for (int e = tid; e < s.E; e += kWideThreads) out_of(nth(k))[e] = from_f<T>(__int_as_float(0x7fffffff));
            if (tid == 0) atomicExch(&g_step_error, 1);
            break;
        }
        // columns' sums, u and o by a thread each, and u for all
        float* us = row + 4 * kMaxStep;
        if (tid < s.E) {
            const float *p = reinterpret_cast<const float*>(part) + tid, *q = p + 4 * kWideThreads;
            float a = 0.f, y = 0.f;
            for (int n = 0; n < R; ++n) {
                a += p[n * s.E];
                y += q[n * s.E];
            }
            const float u = beta * (v - a);
            us[tid] = u;
            o[tid] = from_f<T>(fmaf(qk, u, y) * s.scale);
        }
        workers(true);
        if (busy) {
            const float4 u = *reinterpret_cast<const float4*>(us + 4 * c);
#pragma unroll
            for (int n = 0; n < kWidePer; ++n) {
                const int d = r + n * R;
                if (d >= s.D) break;
                const float kd = sk[d];
                x[n].x = fmaf(kd, u.x, x[n].x);
                x[n].y = fmaf(kd, u.y, x[n].y);
                x[n].z = fmaf(kd, u.z, x[n].z);
                x[n].w = fmaf(kd, u.w, x[n].w);
                S[d * C] = x[n];
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if ((tid & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(done + 8 * place) : "memory");
    }
}

// ---- whole recordings ---------------------------------------------------------------------------------------------------

int size_of(long long type) { return type == FG_F32 ? 4 : 2; }
Operand operand(const fg_ticks& t, long long heads, long long of, long long dim, int size) {
    const long long e = 16 / size;
    const bool fast = dim % 8 == 0 && reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && t.batch % e == 0 && t.tick % e == 0 && t.head % e == 0;
    return {static_cast<char*>(t.p), t.batch, t.tick, t.head, (int)(heads / of), fast};
}
Gate gate(const fg_ticks& t) { return {static_cast<float*>(t.p), t.batch, t.tick, t.head}; }

void check_heads(const std::string& who, long long heads, std::initializer_list<long long> shared) {
    bool ok = heads >= 1 && heads <= 65535;
    for (long long n : shared) ok = ok && n >= 1 && heads % n == 0;
    if (!ok) throw MemErr{who + ": heads must be a multiple of query_heads, key_heads and value_heads, 1 to 65535"};
}
long long slots_of(const fg_delta_args* g) {
    return g->offsets ? g->ticks / kTicks + g->batch : g->batch * ((g->ticks + kTicks - 1) / kTicks);
}
void check_sizes(const fg_delta_args* g, const std::string& who) {
    if (!g) throw MemErr{who + ": no arguments"};
    if (g->batch < 0 || g->ticks < 0) throw MemErr{who + ": a negative size"};
    check_heads(who, g->heads, {g->query_heads, g->key_heads, g->value_heads});
    if (g->dim < 1 || g->dim > kMaxDim || g->value_dim < 1 || g->value_dim > kMaxValue)
        throw MemErr{who + ": dim must be 1 to 128, value_dim 1 to 256"};
    if (g->type < FG_F32 || g->type > FG_F16) throw MemErr{who + ": unknown type"};
    // (each in turn, so that no product overflows)
    const bool few = g->batch <= (1ll << 27) && g->ticks <= (1ll << 36) && g->batch * g->heads <= (1ll << 27) && slots_of(g) <= (1ll << 30) &&
                     slots_of(g) * g->heads <= (1ll << 38);
    if (!few) throw MemErr{who + ": too many recordings or ticks"};
}
long long all_ticks(const fg_delta_args* g) { return g->offsets ? g->ticks : g->batch * g->ticks; }

// The workspace's parts, each from a 256-byte boundary on
struct Room {
    char* p;
    long long used = 0;
    template <class P>
    void take(P*& to, long long bytes) {
        to = p ? reinterpret_cast<P*>(p + used) : nullptr;
        used += (bytes + 255) / 256 * 256;
    }
};
struct Wide {
    float *q = nullptr, *k = nullptr, *v = nullptr;   // gradients of each head in fp32, of shared ones
    bf16 *high = nullptr, *low = nullptr;             // dN as two terms, of 16-bit values that are not shared
};
// Parts of a recording (k_delta_join): as many as keep the blocks within one round of the SMs, of 512 ticks at least; four at least, or
// the work is not worth it. 1 recording of 65,536 ticks, 8 heads of 128 in bf16: 1,310 us in 27 parts
// (the parts' own 709, put together 78, then 522), as many chunks one after another 5,230.
int parts_of(const fg_delta_args* g) {
    const long long rows = std::max<long long>(1, g->batch * g->heads), mean = g->offsets ? g->ticks / std::max<long long>(1, g->batch) : g->ticks;
    const long long parts = std::min<long long>(64, std::min(12 * kSms / (rows * ((g->value_dim + 15) / 16)), mean / 512));
    return parts >= 4 ? (int)parts : 1;
}
// What the way back can take over from the way forward, and what only a call itself needs: `held` and the workspace (g->work), or, without
// a forward that held it, both in the workspace. Returns their sizes.
struct Sizes {
    long long work, held;
};
Sizes lay_out(const fg_delta_args* g, bool backward, bool holds, void* held, Delta& s, Wide& wide) {
    Room room{static_cast<char*>(g->work)}, over{static_cast<char*>(held)};
    Room& kept = holds ? over : room;
    const auto of = [&](auto f) {
        return g->type == FG_F32 ? f(Terms<float>()) : g->type == FG_F16 ? f(Terms<__half>()) : f(Terms<bf16>());
    };
    const bool all_terms = backward || holds;
    const int terms = of([](auto t) { return t.kept; }), out = of([](auto t) { return t.out_p; });
    const long long places = slots_of(g) * g->heads, tiles = (g->value_dim + 15) / 16, padded = g->dim > 64 ? 128 : 64;
    if (g->offsets) kept.take(s.table, slots_of(g) * (long long)sizeof(Slot));
    kept.take(s.x, places * terms * 2 * kChunk * kChunk * 2);
    kept.take(s.p, places * (all_terms ? terms : out) * 2 * kChunk * kChunk * 2);
    kept.take(s.gates, places * kGates * kTicks * 4);
    s.parts = parts_of(g);
    if (s.parts > 1) {
        const long long all = g->batch * g->heads * s.parts * 4, dim = padded;
        room.take(s.own, all * 16 * tiles * dim);
        kept.take(s.turn, all * dim * dim);
        room.take(s.start, all * 16 * tiles * dim);
    }
    if (all_terms) {
        kept.take(s.states, places * tiles * padded * 64);
        kept.take(s.w, places * tiles * 8 * 512);
        kept.take(s.o32, places * tiles * 8 * 512);
        kept.take(s.kept_last, g->batch * g->heads * g->dim * g->value_dim * 4);
    }
    if (backward) {
        room.take(s.gstates, places * tiles * padded * 64);
        room.take(s.od, places * tiles * kTicks * 4);
        room.take(s.vdn, places * tiles * kTicks * 4);
        room.take(s.db, places * tiles * kTicks * 4);
        room.take(s.anchor, places * tiles * 4);
        const long long rows = all_ticks(g) * g->heads * 4;
        if (g->query_heads != g->heads) room.take(wide.q, rows * g->dim);
        if (g->key_heads != g->heads) room.take(wide.k, rows * g->dim);
        if (g->value_heads != g->heads) {
            room.take(wide.v, rows * g->value_dim);
        } else if (g->type != FG_F32) {
            if (g->type == FG_F16) room.take(wide.high, rows / 2 * padded_values((int)g->value_dim));
            room.take(wide.low, rows / 2 * padded_values((int)g->value_dim));
        }
    }
    return {room.used, over.used};
}

void check(const fg_delta_args* g, bool backward, bool holds, const void* held, long long held_bytes) {
    const std::string who = backward ? "fg_delta_attn_bwd" : "fg_delta_attn";
    check_sizes(g, who);
    const auto want = [&](bool ok, const char* what) {
        if (!ok) throw MemErr{who + ": " + what};
    };
    if (g->batch && g->ticks) {
        want(g->q.p && g->k.p && g->v.p && g->log_decay.p && g->beta.p, "null pointer");
        want(backward ? g->go.p && g->gq.p && g->gk.p && g->gv.p && g->glog_decay.p && g->gbeta.p : g->o.p != nullptr, "null pointer");
    }
    want(backward || !g->state || g->state != g->state_out, "state and state_out are the same");
    want(!backward || !g->gstate || (g->gstate != g->state && g->gstate != g->gstate_out), "gstate is state or gstate_out");
    Delta s{};
    Wide wide;
    const Sizes bytes = lay_out(g, backward, holds, nullptr, s, wide);
    want(!bytes.work || (g->work && g->work_bytes >= bytes.work), "the workspace is too small");
    want(reinterpret_cast<uintptr_t>(g->work) % 16 == 0, "the workspace is not 16-byte aligned");
    want(!holds || !bytes.held || (held && held_bytes >= bytes.held), "what is held is too small");
    want(reinterpret_cast<uintptr_t>(held) % 16 == 0, "what is held is not 16-byte aligned");
}

Delta delta_of(const fg_delta_args* g) {
    Delta s{};
    const int size = size_of(g->type);
    s.q = operand(g->q, g->heads, g->query_heads, g->dim, size);
    s.k = operand(g->k, g->heads, g->key_heads, g->dim, size);
    s.v = operand(g->v, g->heads, g->value_heads, g->value_dim, size);
    s.o = operand(g->o, g->heads, g->heads, g->value_dim, size);
    s.go = operand(g->go, g->heads, g->heads, g->value_dim, size);
    s.log_decay = gate(g->log_decay);
    s.beta = gate(g->beta);
    s.first = g->state;
    s.last = g->state_out;
    s.offsets = g->offsets;
    s.batch = g->batch;
    s.ticks = g->ticks;
    s.slots = slots_of(g);
    s.heads = (int)g->heads;
    s.D = (int)g->dim;
    s.E = (int)g->value_dim;
    s.scale = (float)g->scale;
    return s;
}

template <class K>
void launch(K* kernel, dim3 grid, int threads, int bytes, OnEachDevice& here, cudaStream_t st, const Delta& s) {
    here.first(current_device(), [&] { allow_shared(kernel, bytes); });
    kernel<<<grid, threads, bytes, st>>>(s);
    MCK(cudaGetLastError());
}
template <class T, int DP, int NP>
void prepare(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    if (s.offsets && s.slots) {
        k_delta_slots<<<(unsigned)((s.slots + 127) / 128), 128, 0, st>>>(s);
        MCK(cudaGetLastError());
    }
    if (s.slots) launch(k_delta_prep<T, DP, NP>, dim3((unsigned)s.slots, s.heads), 128, PrepLayout<T, DP>::bytes, here, st, s);
}
// WARPS: 16 columns of values each
template <class T, int DP, int WARPS, int MODE>
void chain(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    using Lay = ChainLayout<T, DP, WARPS, MODE == kKeep ? Terms<T>::kept : Terms<T>::out_p, MODE == kKeep>;
    const int tiles = (s.E + 15) / 16 + (MODE == kParts ? (s.D + 15) / 16 : 0);
    const long long blocks = s.batch * s.heads * ((tiles + WARPS - 1) / WARPS);
    launch(k_delta_chain<T, DP, WARPS, MODE>, dim3((unsigned)blocks, s.parts), 32 * WARPS, Lay::bytes, here, st, s);
}
template <class T, int DP, int WARPS, bool PARTS>
void chain_back(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    const long long blocks = s.batch * s.heads * ((s.E + 16 * WARPS - 1) / (16 * WARPS));
    launch(k_delta_back<T, DP, WARPS, PARTS>, dim3((unsigned)blocks, s.parts), 32 * WARPS, ChainLayout<T, DP, WARPS, Terms<T>::kept, true>::bytes,
           here, st, s);
}
template <int DP, bool BACK>
void join(const Delta& s, cudaStream_t st) {
    k_delta_join<DP, BACK><<<(unsigned)(s.batch * s.heads * ((s.E + 15) / 16)), 2 * DP, 0, st>>>(s);
    MCK(cudaGetLastError());
}
template <class T>
void gradients(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    if (s.slots) launch(k_delta_grads<T>, dim3((unsigned)s.slots, s.heads, (s.D + 63) / 64), 256, GradLayout<T>::bytes, here, st, s);
}

// the state that each part of a recording begins with
template <class T, int DP>
void parts_forward(const Delta& s, cudaStream_t st) {
    if (s.parts == 1) return;
    chain<T, DP, 4, kParts>(s, st);
    join<DP, false>(s, st);
}
// forward, and all that the way back needs
// 64 or 128 columns of values a block: 16 warps an SM with 128 registers a thread where dim is over 64 (forward and back 800 and 1,015 us;
// before O was kept 777 and 917, where blocks of 4 warps with 168 registers took 1,185 and 1,030)
template <class T, int DP>
constexpr int wide_block = Terms<T>::in == 1 && DP == 128 ? 8 : 4;
template <class T, int DP>
void forward_kept(const Delta& s, cudaStream_t st) {
    prepare<T, DP, Terms<T>::kept>(s, st);
    parts_forward<T, DP>(s, st);
    if (s.E > 64) chain<T, DP, wide_block<T, DP>, kKeep>(s, st);
    else chain<T, DP, 4, kKeep>(s, st);
}
template <class T, int DP>
void forward(const Delta& s, bool keep, cudaStream_t st) {
    if (keep) return forward_kept<T, DP>(s, st);
    prepare<T, DP, Terms<T>::out_p>(s, st);
    parts_forward<T, DP>(s, st);
    chain<T, DP, 4, kForward>(s, st);
}
template <class T, int DP>
void backward(const Delta& s, bool kept, cudaStream_t st) {
    if (!kept) forward_kept<T, DP>(s, st);
    if (s.parts > 1) {
        chain_back<T, DP, 4, true>(s, st);
        join<DP, true>(s, st);
    }
    if (s.E > 64) chain_back<T, DP, wide_block<T, DP>, false>(s, st);
    else chain_back<T, DP, 4, false>(s, st);
    gradients<T>(s, st);
}

int attn(const fg_delta_args* g, bool holds, void* held, long long held_bytes, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, false, holds, held, held_bytes);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        clear_outside(g->offsets, g->batch, g->ticks, {&g->o}, {g->heads}, {g->value_dim}, 1, size_of(g->type), st);
        if (!g->batch) return 0;
        Delta s = delta_of(g);
        Wide wide;
        lay_out(g, false, holds, held, s, wide);
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            if (s.D > 64) forward<T, 128>(s, holds, st);
            else forward<T, 64>(s, holds, st);
        });
        return 0;
    });
}

int attn_bwd(const fg_delta_args* g, bool holds, void* held, long long held_bytes, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, true, holds, held, held_bytes);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const auto clear = [&] {                              // (last: sums of shared heads go over all ticks)
            clear_outside(g->offsets, g->batch, g->ticks, {&g->gq, &g->gk, &g->gv}, {g->query_heads, g->key_heads, g->value_heads},
                          {g->dim, g->dim, g->value_dim}, 3, size_of(g->type), st);
            clear_outside(g->offsets, g->batch, g->ticks, {&g->glog_decay, &g->gbeta}, {g->heads, g->heads}, {1, 1}, 2, 4, st);
        };
        if (!g->batch) {
            clear();
            return 0;
        }
        Delta s = delta_of(g);
        Wide wide;
        lay_out(g, true, holds, held, s, wide);
        s.o.p = nullptr;
        s.last = nullptr;
        s.glast = g->gstate_out;
        s.gfirst = g->gstate;
        s.glog_decay = gate(g->glog_decay);
        s.gbeta = gate(g->gbeta);
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            // gradients of shared heads: of each head in fp32, then added
            const auto out = [&](Operand& to, int& f32, const fg_ticks& o, float* room, long long dim) {
                const fg_ticks all{room, g->ticks * g->heads * dim, g->heads * dim, dim};
                f32 = room || std::is_same<T, float>::value;
                to = operand(room ? all : o, g->heads, g->heads, dim, f32 ? 4 : (int)sizeof(T));
            };
            out(s.gq, s.gq_f32, g->gq, wide.q, g->dim);
            out(s.gk, s.gk_f32, g->gk, wide.k, g->dim);
            out(s.dn, s.dn_f32, g->gv, wide.v, g->value_dim);
            const auto term = [&](Operand& to, bf16* room) {
                const long long row = padded_values(s.E);
                to = operand({room, g->ticks * g->heads * row, g->heads * row, row}, g->heads, g->heads, row, 2);
            };
            term(s.dn_low, wide.low);
            if (std::is_same<T, bf16>::value) s.dn_high = s.dn;
            else term(s.dn_high, wide.high);
            if (s.D > 64) backward<T, 128>(s, holds, st);
            else backward<T, 64>(s, holds, st);
            const auto add = [&](const fg_ticks& to, long long heads, long long dim, const float* room) {
                if (room && all_ticks(g))
                    share_sum<T>(room, to, g->offsets ? 1 : g->batch, g->ticks, (int)g->heads, (int)heads, (int)dim, st);
            };
            add(g->gq, g->query_heads, g->dim, wide.q);
            add(g->gk, g->key_heads, g->dim, wide.k);
            add(g->gv, g->value_heads, g->value_dim, wide.v);
        });
        clear();
        return 0;
    });
}

}  // namespace

extern "C" {

static Sizes delta_sizes(const fg_delta_args* g, const char* who, bool backward, bool holds) {
    check_sizes(g, who);
    fg_delta_args sizes = *g;
    sizes.work = nullptr;
    Delta s{};
    Wide wide;
    return lay_out(&sizes, backward, holds, nullptr, s, wide);
}
long long fg_delta_work(const fg_delta_args* g, int backward) {
    return mem_guard([&]() -> long long { return delta_sizes(g, "fg_delta_work", backward & 1, backward >> 1 & 1).work; });
}
long long fg_delta_held(const fg_delta_args* g) {
    return mem_guard([&]() -> long long { return delta_sizes(g, "fg_delta_held", false, true).held; });
}

int fg_delta_attn(const fg_delta_args* g, void* stream) { return attn(g, false, nullptr, 0, stream); }
int fg_delta_attn_hold(const fg_delta_args* g, void* held, long long held_bytes, void* stream) { return attn(g, true, held, held_bytes, stream); }
int fg_delta_attn_bwd(const fg_delta_args* g, void* stream) { return attn_bwd(g, false, nullptr, 0, stream); }
int fg_delta_attn_bwd_held(const fg_delta_args* g, void* held, long long held_bytes, void* stream) {
    return attn_bwd(g, true, held, held_bytes, stream);
}

int fg_delta_step(const fg_delta_step_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        const std::string who = "fg_delta_step";
        need(g, "fg_delta_step: no arguments");
        need(g->batch >= 0 && g->n_slots >= 0, "fg_delta_step: a negative size");
        check_heads(who, g->heads, {g->query_heads, g->key_heads, g->value_heads});
        need(g->dim >= 1 && g->dim <= kMaxStep && g->value_dim >= 1 && g->value_dim <= kMaxStep, "fg_delta_step: dim and value_dim must be 1 to 256");
        need(g->batch * g->heads <= (1ll << 27) && g->batch <= (1ll << 27), "fg_delta_step: batch * heads is over 2^27");
        need(g->type >= FG_F32 && g->type <= FG_F16, "fg_delta_step: unknown type");
        if (!g->batch) return 0;
        need(g->q.p && g->k.p && g->v.p && g->o.p && g->log_decay.p && g->beta.p && (g->state || !g->n_slots), "fg_delta_step: null pointer");
        Step s{};
        s.q = g->q, s.k = g->k, s.v = g->v, s.o = g->o;
        s.log_decay = static_cast<const float*>(g->log_decay.p);
        s.beta = static_cast<const float*>(g->beta.p);
        s.log_batch = g->log_decay.batch, s.log_head = g->log_decay.head;
        s.beta_batch = g->beta.batch, s.beta_head = g->beta.head;
        s.state = g->state;
        s.slots = g->slots;
        s.n_slots = g->n_slots;
        s.heads = (int)g->heads;
        s.q_share = (int)(g->heads / g->query_heads);
        s.k_share = (int)(g->heads / g->key_heads);
        s.v_share = (int)(g->heads / g->value_heads);
        s.D = (int)g->dim;
        s.E = (int)g->value_dim;
        s.tiles = (s.E + 31) / 32;
        s.scale = (float)g->scale;
        const bool by4 = g->value_dim % 4 == 0 && reinterpret_cast<uintptr_t>(g->state) % 16 == 0;
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            const long long items = g->batch * g->heads;
            // whole states through shared memory where each SM has several (2,048 rows, 8 heads of 128 x 128: 476 us by columns)
            if (by4 && items >= 8 * kSms && s.D * s.E <= 16384 && s.D <= kWidePer * (kWideThreads / (s.E / 4))) {
                const int bytes = WideLayout(s.D, s.E).bytes;
                static OnEachDevice here;
                here.first(current_device(), [] { allow_shared(k_delta_step_wide<T>, WideLayout(128, 128).bytes); });
                k_delta_step_wide<T><<<kSms, kWideThreads + 32, bytes, static_cast<cudaStream_t>(stream)>>>(s, (uint32_t)items);
                return;
            }
            auto* kernel = by4 ? s.D <= 64 ? k_delta_step<T, 4, 2> : s.D <= 128 ? k_delta_step<T, 4, 4> : k_delta_step<T, 4, 8>
                               : s.D <= 64 ? k_delta_step<T, 1, 8> : k_delta_step<T, 1, 32>;
            kernel<<<(unsigned)(g->batch * g->heads * s.tiles), 256, 0, static_cast<cudaStream_t>(stream)>>>(s);
        });
        MCK(cudaGetLastError());
        return 0;
    });
}

}  // extern "C"

namespace fgm {
int step_gave_up(cudaStream_t st) {
    int bad = 0;
    MCK(cudaMemcpyFromSymbolAsync(&bad, g_step_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
    MCK(cudaStreamSynchronize(st));
    return bad;
}
}  // namespace fgm
