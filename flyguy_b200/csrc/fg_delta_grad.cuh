// The gradients of q, k and the gates, every slot of 64 ticks by itself (a chunk as in fg_delta_chain.cuh, of 64: the same formulas), from
// what the chain forward (S before the slot, W) and the chain back (R behind it, dN, rows of dots) have left:
//
//   dP = dO U^T . M on and below the diagonal, D = -dN U^T . M below it
//   dQ = scale (e^G dO S^T + dP K),  dK = scale dP^T Q + (D + D^T) K - e^G dN S^T + e^{G_63 - G} U R^T
//   dbeta: the tiles' rows added;  dlog_decay_t = <R, S> + sum over t' >= t of (o dO - v dN)_t'
//
// A block of 8 warps makes 64 columns of one slot of one head: warp = 16 ticks x 32 columns. The products with S and R run over blocks of 64
// of their columns; S, R and W arrive as the chain's accumulators and go through shared memory, where reading across turns them.
//
// 64 recordings of 1,024 ticks, 8 heads of 128 in bf16: 1,032 us (2.3 GB, 350 us at a plain copy's rate; the products 440). Bound by what follows one
// another in a block of which an SM holds two: the loads, their terms, the products, the masks; tensor pipe 42%, issue slots 36%, DRAM 33%.
#pragma once
#include "fg_delta_chain.cuh"

namespace {

template <class T>
struct GradLayout {
    static constexpr int in = Terms<T>::in, terms_n = Terms<T>::grad_n, terms_s = Terms<T>::grad_s, terms_r = Terms<T>::grad_r, terms = Terms<T>::grad, plane = kTicks * kSquare;
    static constexpr int q = 0, k = q + in * plane, go = k + in * plane, dn = go + in * plane, u = dn + terms_n * plane, s = u + terms * plane,
                         r = s + terms_s * plane, values = r + terms_r * plane;
    static constexpr int dp = go, d = dp + terms * plane;     // later, over dO, dN and U
    static constexpr int out = s;                             // and at last, fp32 rows over S and R
    static constexpr int bytes = 2 * values + 4 * kGates * kTicks;
    static_assert(terms_s >= terms_r && in + terms_n >= terms && (terms_s + terms_r) * plane >= 2 * kTicks * 68 && bytes <= 227 * 1024, "room");
};

template <class T>
__global__ void __launch_bounds__(256, Terms<T>::in == 1 ? 2 : 1) k_delta_grads(const __grid_constant__ Delta s) {
    using Lay = GradLayout<T>;
    constexpr int NI = Lay::in, NN = Lay::terms_n, NS = Lay::terms_s, NR = Lay::terms_r, NG = Lay::terms, kPlane = Lay::plane;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* tiles = reinterpret_cast<bf16*>(smem);
    float* gates = reinterpret_cast<float*>(smem + 2 * Lay::values);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const long long slot = blockIdx.x, place = slot * s.heads + blockIdx.y;
    const int h = blockIdx.y, d_block = 64 * blockIdx.z, tiles_e = (s.E + 15) / 16;
    const int padded_d = s.D > 64 ? 16 : 8;                  // the chain's 8-value pieces of a column
    const Slot c = ticks_of(s, slot);
    if (c.n == 0) return;
    const long long tick = c.tick;
    const T* go_rows = row_of<const T>(s, s.go, c.b, h, tick);
    const float* dn_rows = s.dn_f32 ? row_of<const float>(s, s.dn, c.b, h, tick) : nullptr;
    const bf16 *dn_high = s.dn_f32 ? nullptr : row_of<const bf16>(s, s.dn_high, c.b, h, tick),
               *dn_low = s.dn_f32 ? nullptr : row_of<const bf16>(s, s.dn_low, c.b, h, tick);
    const int wt = warp >> 1, wd = warp & 1;                 // ticks 16 wt .., columns (of d, or ticks s) 32 wd ..

    load_tile<T, NI, 64, kSquare, 256>(tiles + Lay::q, row_of<const T>(s, s.q, c.b, h, tick) + d_block, s.q.tick, c.n, s.D - d_block, s.q.fast, tid);
    load_tile<T, NI, 64, kSquare, 256>(tiles + Lay::k, row_of<const T>(s, s.k, c.b, h, tick) + d_block, s.k.tick, c.n, s.D - d_block, s.k.fast, tid);
    for (int i = tid; i < kGates * kTicks; i += 256) gates[i] = s.gates[place * kGates * kTicks + i];

    float dq[4][4] = {}, dk[4][4] = {}, du[4][4] = {}, dp[4][4] = {}, dd[4][4] = {};
    const uint32_t at_m = smem_at(tiles) + at_rows_m(lane, kSquare), at_n = smem_at(tiles) + at_rows_n(lane, kSquare);
    const bool below = 32 * wd <= 16 * wt;                   // this warp's ticks s x t meet the diagonal's lower side
    const float* beta = s.gates + (place * kGates + 2) * kTicks;
    if (lane < 16 && (warp >> 1) < tiles_e) prefetch(reinterpret_cast<const char*>(s.w + ((2 * place + (warp & 1)) * tiles_e + (warp >> 1)) * 4 * 32) + lane * 128);
#pragma unroll 1
    for (int e0 = 0; e0 < s.E; e0 += 64) {
        if (e0) __syncthreads();
        load_tile<T, NI, 64, kSquare, 256>(tiles + Lay::go, go_rows + e0, s.go.tick, c.n, s.E - e0, s.go.fast, tid);
        if (s.dn_f32)
            load_tile<float, NN, 64, kSquare, 256>(tiles + Lay::dn, dn_rows + e0, s.dn.tick, c.n, s.E - e0, s.dn.fast, tid);
        else if constexpr (sizeof(T) == 2) {
            static_assert(NN == 2, "dN's terms");
            const int whole = padded_values(s.E) - e0;
            load_tile<bf16, 1, 64, kSquare, 256>(tiles + Lay::dn, dn_high + e0, s.dn_high.tick, c.n, std::is_same<T, bf16>::value ? s.E - e0 : whole,
                                                 s.dn_high.fast, tid);
            load_tile<bf16, 1, 64, kSquare, 256>(tiles + Lay::dn + kPlane, dn_low + e0, s.dn_low.tick, c.n, whole, s.dn_low.fast, tid);
        }
        async_commit();
        if (e0 + 64 < s.E) {                                  // the next columns on their way to L2
            const int e = e0 / 16 + 4 + (warp >> 1);
            if (e < tiles_e) {
                prefetch(reinterpret_cast<const char*>((warp & 1 ? s.gstates : s.states) + ((place * tiles_e + e) * padded_d + d_block / 8) * 32) + lane * 128);
                if (lane < 16) prefetch(reinterpret_cast<const char*>(s.w + ((2 * place + (warp & 1)) * tiles_e + e) * 4 * 32) + lane * 128);
            }
            const int row = tid & 63, which = tid >> 6;
            const void* rows[3] = {go_rows + row * s.go.tick + e0 + 64, dn_high + row * s.dn_high.tick + e0 + 64, dn_low + row * s.dn_low.tick + e0 + 64};
            if (s.dn_f32) rows[1] = rows[2] = dn_rows + row * s.dn.tick + e0 + 64;
            if (which < (s.dn_f32 ? 2 : 3) && row < c.n) prefetch(static_cast<const char*>(rows[which]));
        }
        // S and R, accumulators of 16 columns x 8 values -> terms in rows of columns; a warp: 16 columns of one of them
        {
            const int which = warp & 1, te = warp >> 1, e = e0 / 16 + te;
            const float4* from = (which ? s.gstates : s.states) + ((place * tiles_e + e) * padded_d + d_block / 8) * 32 + lane;
            const uint32_t to = smem_at(tiles) + 2 * ((which ? Lay::r : Lay::s) + 16 * te * kSquare) + at_rows_m(lane, kSquare);
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = e < tiles_e ? __ldg(from + j * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a[NS][4];
                const float x[2][4] = {{v[2 * j].x, v[2 * j].y, v[2 * j].z, v[2 * j].w}, {v[2 * j + 1].x, v[2 * j + 1].y, v[2 * j + 1].z, v[2 * j + 1].w}};
                left<NS>(x[0], x[1], a);
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    if (which && n >= NR) break;
                    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(to + 2 * (n * kPlane + 16 * j)), "r"(a[n][0]),
                                 "r"(a[n][1]), "r"(a[n][2]), "r"(a[n][3])
                                 : "memory");
                }
            }
        }
        // U = B W; a warp: 16 columns of one chunk (without ticks: zeros)
        {
            const int te = warp >> 1, half = warp & 1, e = e0 / 16 + te;
            const bool there = e < tiles_e && (half == 0 || c.n > kChunk);
            const float4* from = s.w + ((2 * place + half) * tiles_e + e) * 4 * 32 + lane;
            const uint32_t to = smem_at(tiles) + 2 * (Lay::u + 32 * half * kSquare + 16 * te) + at_rows_n(lane, kSquare);
            float4 v[4];
            float2 by[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = there ? __ldg(from + j * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
                by[j] = __ldg(reinterpret_cast<const float2*>(beta + 32 * half + 8 * j + 2 * t4));
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x[2][4] = {{v[2 * j].x, v[2 * j].y, v[2 * j].z, v[2 * j].w}, {v[2 * j + 1].x, v[2 * j + 1].y, v[2 * j + 1].z, v[2 * j + 1].w}};
#pragma unroll
                for (int i = 0; i < 2; ++i) scale2(x[i], by[2 * j + i]);
                uint32_t a[NG][4];
                left<NG>(x[0], x[1], a);
#pragma unroll
                for (int n = 0; n < NG; ++n) stsm_t(to + 2 * (n * kPlane + 16 * j * kSquare), a[n]);
            }
        }
        async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t go[NI][4], dn[NN][4], u[NG][4];
#pragma unroll
            for (int n = 0; n < NI; ++n) ldsm(go[n], at_m + 2 * (Lay::go + n * kPlane + 16 * wt * kSquare + 16 * e));
#pragma unroll
            for (int n = 0; n < NN; ++n) ldsm(dn[n], at_m + 2 * (Lay::dn + n * kPlane + 16 * wt * kSquare + 16 * e));
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                ldsm(u[n], at_m + 2 * (Lay::u + n * kPlane + 16 * wt * kSquare + 16 * e));
            }
            const auto state = [&](int j, int p) { return at_m + 2 * (Lay::s + j * kPlane + 16 * e * kSquare + 32 * wd + 16 * p); };
            products<NI, NS, NG, 2, true>(dq, go, state);
            products<NN, NS, NG, 2, true>(dk, dn, state);
            products<NG, NR, NG, 2, true>(du, u, [&](int j, int p) { return at_m + 2 * (Lay::r + j * kPlane + 16 * e * kSquare + 32 * wd + 16 * p); });
            if (below) {
                const auto at = [&](int j, int p) { return at_n + 2 * (Lay::u + j * kPlane + (32 * wd + 16 * p) * kSquare + 16 * e); };
                products<NI, NG, NG, 2, false>(dp, go, at);
                products<NN, NG, NG, 2, false>(dd, dn, at);
            }
        }
    }
    __syncthreads();                                          // dO, dN, U, S and R have been read
    const float *gh = gates + 3 * kTicks, *gl = gates + 4 * kTicks;
    if (below) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = 16 * wt + g + 8 * i, c0 = 32 * wd + 8 * j + 2 * t4;
                float x[2], y[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = t >= c0 + e ? expf((gh[t] - gh[c0 + e]) + (gl[t] - gl[c0 + e])) : 0.f;
                    x[e] = t >= c0 + e ? dp[j][2 * i + e] * (f * s.scale) : 0.f;
                    y[e] = t > c0 + e ? -dd[j][2 * i + e] * f : 0.f;
                }
                uint32_t a[NG], b[NG];
                terms<NG>(x[0], x[1], a);
                terms<NG>(y[0], y[1], b);
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    *reinterpret_cast<uint32_t*>(tiles + Lay::dp + n * kPlane + t * kSquare + c0) = a[n];
                    *reinterpret_cast<uint32_t*>(tiles + Lay::d + n * kPlane + t * kSquare + c0) = b[n];
                }
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = 16 * wt + g + 8 * i;
        const float f = expf(gh[t] + gl[t]), k = expf((gh[kTicks - 1] - gh[t]) + (gl[kTicks - 1] - gl[t]));
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; ++e) {
                dq[j][e] *= f * s.scale;
                dk[j][e] = fmaf(-f, dk[j][e], k * du[j][e]);
            }
    }
    __syncthreads();
    // rows of dP and D by K; columns of dP by Q, of D by K
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t a[NG][4], b[NG][4];
        const auto keys = [&](int j, int p) { return at_m + 2 * (Lay::k + j * kPlane + 16 * k * kSquare + 32 * wd + 16 * p); };
        if (k <= wt) {
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                ldsm(a[n], at_m + 2 * (Lay::dp + n * kPlane + 16 * wt * kSquare + 16 * k));
                ldsm(b[n], at_m + 2 * (Lay::d + n * kPlane + 16 * wt * kSquare + 16 * k));
            }
            products<NG, NI, NG, 2, true>(dq, a, keys);
            products<NG, NI, NG, 2, true>(dk, b, keys);
        }
        if (k >= wt) {
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                ldsm_t(a[n], at_n + 2 * (Lay::dp + n * kPlane + 16 * k * kSquare + 16 * wt));
                ldsm_t(b[n], at_n + 2 * (Lay::d + n * kPlane + 16 * k * kSquare + 16 * wt));
            }
            products<NG, NI, NG, 2, true>(dk, a, [&](int j, int p) { return at_m + 2 * (Lay::q + j * kPlane + 16 * k * kSquare + 32 * wd + 16 * p); });
            products<NG, NI, NG, 2, true>(dk, b, keys);
        }
    }
    // by way of shared memory (over S and R), so that a row leaves in whole sectors
    float* stage = reinterpret_cast<float*>(tiles + Lay::out);
    constexpr int kRow = 68;
    const auto put = [&](const Operand& o, int f32, const float (&x)[4][4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *reinterpret_cast<float2*>(stage + (16 * wt + g + 8 * i) * kRow + 32 * wd + 8 * j + 2 * t4) = make_float2(x[j][2 * i], x[j][2 * i + 1]);
        __syncthreads();
        const int r0 = tid >> 3, col = (tid & 7) * 8, d = d_block + col;
        const long long at = (s.offsets ? 0 : (long long)c.b * o.batch) + tick * o.tick + h * o.head + d;   // (gradients of each head by itself)
        if (d < s.D) {
#pragma unroll
            for (int r = r0; r < kTicks; r += 32) {
                if (r >= c.n) break;
                float v[8];
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(stage + r * kRow + col);
                *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(stage + r * kRow + col + 4);
                if (f32) {
                    float* to = reinterpret_cast<float*>(o.p) + at + r * o.tick;
                    if (o.fast) {
                        reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
                        reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
                        for (int j = 0; j < 8 && d + j < s.D; ++j) to[j] = v[j];
                    }
                } else if constexpr (sizeof(T) == 2) {
                    T* to = reinterpret_cast<T*>(o.p) + at + r * o.tick;
                    T w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = from_f<T>(v[j]);
                    if (o.fast) {
                        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(w);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (d + j < s.D) to[j] = w[j];
                    }
                }
            }
        }
    };
    put(s.gq, s.gq_f32, dq);
    __syncthreads();
    put(s.gk, s.gk_f32, dk);
    // the gates' gradients
    if (blockIdx.z == 0 && warp == 0) {
        float dot[2] = {}, db[2] = {}, anchor = 0.f;
        for (int e = 0; e < tiles_e; ++e) {
            const long long at = (place * tiles_e + e) * kTicks + 2 * lane;
            const float2 o = *reinterpret_cast<const float2*>(s.od + at), v = *reinterpret_cast<const float2*>(s.vdn + at),
                         x = *reinterpret_cast<const float2*>(s.db + at);
            dot[0] += o.x - v.x;
            dot[1] += o.y - v.y;
            db[0] += x.x;
            db[1] += x.y;
            anchor += s.anchor[place * tiles_e + e];
        }
        float after = dot[0] + dot[1];                       // of this lane's ticks and all later ones
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float x = __shfl_down_sync(0xffffffffu, after, o);
            if (lane + o < 32) after += x;
        }
        const float next = __shfl_down_sync(0xffffffffu, after, 1);
        const float rest = (lane < 31 ? next : 0.f) + anchor;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = 2 * lane + i;
            if (t >= c.n) continue;
            *gate_of(s, s.glog_decay, c.b, h, tick + t) = i ? rest + dot[1] : rest + dot[1] + dot[0];
            *gate_of(s, s.gbeta, c.b, h, tick + t) = db[i];
        }
    }
}

}  // namespace
