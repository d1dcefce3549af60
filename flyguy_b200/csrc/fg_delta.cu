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
// pass over them gives k S and q S, and o = q S + (q k) u needs no second one. State in and out is the cost.
template <class T, int V>
__global__ void __launch_bounds__(256) k_delta_step(const __grid_constant__ Step s) {
    constexpr int kAcross = 32 / V, kRows = 256 / kAcross, kPer = kMaxStep / kRows;
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
void check_sizes(const fg_delta_args* g, const std::string& who) {
    if (!g) throw MemErr{who + ": no arguments"};
    if (g->batch < 0 || g->ticks < 0) throw MemErr{who + ": a negative size"};
    check_heads(who, g->heads, {g->query_heads, g->key_heads, g->value_heads});
    if (g->dim < 1 || g->dim > kMaxDim || g->value_dim < 1 || g->value_dim > kMaxValue)
        throw MemErr{who + ": dim must be 1 to 128, value_dim 1 to 256"};
    if (g->type < FG_F32 || g->type > FG_F16) throw MemErr{who + ": unknown type"};
    if (g->batch * g->heads > (1ll << 27) || g->ticks > (1ll << 36) || g->batch > (1ll << 27)) throw MemErr{who + ": too many recordings or ticks"};
}
long long slots_of(const fg_delta_args* g) {
    return g->offsets ? g->ticks / kTicks + g->batch : g->batch * ((g->ticks + kTicks - 1) / kTicks);
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
    float *q = nullptr, *k = nullptr, *v = nullptr, *last = nullptr;
};
// places s's parts; returns their size
long long lay_out(const fg_delta_args* g, bool backward, Delta& s, Wide& wide) {
    Room room{static_cast<char*>(g->work)};
    const int in = g->type == FG_F32 ? 3 : g->type == FG_F16 ? 2 : 1, kept = std::max(in, 2);
    const long long places = slots_of(g) * g->heads, tiles = (g->value_dim + 15) / 16, pieces = g->dim > 64 ? 8 : 4;
    room.take(s.x, places * kept * kTicks * kTicks * 2);
    room.take(s.p, places * (backward ? kept : in) * kTicks * kTicks * 2);
    room.take(s.gates, places * kGates * kTicks * 4);
    if (!backward) return room.used;
    room.take(s.states, places * tiles * kept * pieces * 512);
    room.take(s.gstates, places * tiles * (in == 1 ? 1 : kept) * pieces * 512);
    room.take(s.w, places * tiles * 8 * 512);
    room.take(s.u, places * kTicks * 16 * tiles * (in == 1 ? 2 : 4));
    room.take(s.od, places * tiles * kTicks * 4);
    room.take(s.vdn, places * tiles * kTicks * 4);
    room.take(s.db, places * tiles * kTicks * 4);
    room.take(s.anchor, places * tiles * 4);
    room.take(wide.last, g->batch * g->heads * g->dim * g->value_dim * 4);
    const long long rows = all_ticks(g) * g->heads * 4;
    if (g->query_heads != g->heads) room.take(wide.q, rows * g->dim);
    if (g->key_heads != g->heads) room.take(wide.k, rows * g->dim);
    if (g->value_heads != g->heads) room.take(wide.v, rows * g->value_dim);
    return room.used;
}

void check(const fg_delta_args* g, bool backward) {
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
    const long long bytes = lay_out(g, backward, s, wide);
    want(!bytes || (g->work && g->work_bytes >= bytes), "the workspace is too small");
    want(reinterpret_cast<uintptr_t>(g->work) % 16 == 0, "the workspace is not 16-byte aligned");
    want(slots_of(g) < (1ll << 31) && g->batch * g->heads * ((g->value_dim + 31) / 32) < (1ll << 31), "too many recordings or ticks");
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
    if (s.slots) launch(k_delta_prep<T, DP, NP>, dim3((unsigned)s.slots, s.heads), 128, PrepLayout<T, DP>::bytes, here, st, s);
}
// WARPS: 16 columns of values each
template <class T, int DP, int WARPS, bool KEEP>
void chain(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    using Lay = ChainLayout<T, DP, WARPS, KEEP ? Terms<T>::kept : Terms<T>::out, KEEP>;
    const long long blocks = s.batch * s.heads * ((s.E + 16 * WARPS - 1) / (16 * WARPS));
    launch(k_delta_chain<T, DP, WARPS, KEEP>, dim3((unsigned)blocks), 32 * WARPS, Lay::bytes, here, st, s);
}
template <class T, int DP, int WARPS>
void chain_back(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    const long long blocks = s.batch * s.heads * ((s.E + 16 * WARPS - 1) / (16 * WARPS));
    launch(k_delta_back<T, DP, WARPS>, dim3((unsigned)blocks), 32 * WARPS, ChainLayout<T, DP, WARPS, Terms<T>::kept, true>::bytes, here, st, s);
}
template <class T>
void gradients(const Delta& s, cudaStream_t st) {
    static OnEachDevice here;
    if (s.slots) launch(k_delta_grads<T>, dim3((unsigned)s.slots, s.heads, (s.D + 63) / 64), 256, GradLayout<T>::bytes, here, st, s);
}

template <class T, int DP>
void forward(const Delta& s, cudaStream_t st) {
    prepare<T, DP, Terms<T>::out>(s, st);
    if constexpr (Terms<T>::in == 1) {
        if (s.E > 64) return chain<T, DP, 8, false>(s, st);
    }
    chain<T, DP, 4, false>(s, st);
}
template <class T, int DP>
void backward(Delta s, float* last, cudaStream_t st) {
    prepare<T, DP, Terms<T>::kept>(s, st);
    s.last = last;
    constexpr bool wide = Terms<T>::in == 1;
    if (wide && s.E > 64) {
        if constexpr (wide) {
            chain<T, DP, 8, true>(s, st);
            chain_back<T, DP, 8>(s, st);
        }
    } else {
        chain<T, DP, 4, true>(s, st);
        chain_back<T, DP, 4>(s, st);
    }
    gradients<T>(s, st);
}

}  // namespace

extern "C" {

long long fg_delta_work(const fg_delta_args* g, int backward) {
    return mem_guard([&]() -> long long {
        check_sizes(g, "fg_delta_work");
        fg_delta_args sizes = *g;
        sizes.work = nullptr;
        Delta s{};
        Wide wide;
        return lay_out(&sizes, backward != 0, s, wide);
    });
}

int fg_delta_attn(const fg_delta_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, false);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        clear_outside(g->offsets, g->batch, g->ticks, {&g->o}, {g->heads}, {g->value_dim}, 1, size_of(g->type), st);
        if (!g->batch) return 0;
        Delta s = delta_of(g);
        Wide wide;
        lay_out(g, false, s, wide);
        by_type(g->type, [&](auto t) {
            using T = decltype(t);
            if (s.D > 64) forward<T, 128>(s, st);
            else forward<T, 64>(s, st);
        });
        return 0;
    });
}

int fg_delta_attn_bwd(const fg_delta_args* g, void* stream) {
    return (int)mem_guard([&]() -> long long {
        check(g, true);
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
        lay_out(g, true, s, wide);
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
            if (s.D > 64) backward<T, 128>(s, wide.last, st);
            else backward<T, 64>(s, wide.last, st);
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
            auto* kernel = by4 ? k_delta_step<decltype(t), 4> : k_delta_step<decltype(t), 1>;
            kernel<<<(unsigned)(g->batch * g->heads * s.tiles), 256, 0, static_cast<cudaStream_t>(stream)>>>(s);
        });
        MCK(cudaGetLastError());
        return 0;
    });
}

}  // extern "C"
