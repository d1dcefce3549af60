// The decay scan of bf16 operands on the tensor cores (tcgen05 kind::f16, accumulators in TMEM), chunks of 128 ticks:
//
//   out_t = scale_out (gamma^{t+1} a_t S + sum_{s<=t} gamma^{t-s} (a_t b_s) c_s)      t, s: ticks of the chunk
//   S    <- gamma^n S + scale_in sum_s gamma^{n-1-s} b_s c_s^T                         n: ticks of the chunk
//
// (run from the back: s >= t, gamma^{s-t}, exponents mirrored). Four products a chunk:
//   A  [128 x 128] = a b^T                operands as they arrive, exact products
//   O1 [128 x E]   = a S                  S rounded to bf16
//   O2 [128 x E]   = (A . gamma^{t-s}) c  the weights as two bf16 terms (2^-17), read from TMEM as the A operand
//   dS [D x E]     = b'^T c               b' = gamma^{n-1-s} b as two bf16 terms, written over b (and a, which O1 is done with)
// S itself stays in fp32 registers for the whole recording: thread = row, so the state is as good as its sums. The one
// rounding to bf16, of S in O1, is of the size of the rounding of out itself.
//
// All operands lie in shared memory without a swizzle, 8 rows x 16 bytes (8 values of one tick) to a core matrix: read
// along the ticks or along the values that is the K-major or the MN-major form of the same bytes, so nothing is
// transposed. a, b, c arrive by 16-byte asynchronous copies (zero-filled past the recording's end) a chunk ahead of
// their use. 8 warps; warps w and w + 4 share the TMEM lanes 32 (w % 4) .. and take alternate blocks of 16 columns.
#pragma once
#include "fg_memory.cuh"
#include "fg_tcgen05.cuh"

namespace {
using namespace fgm;

constexpr int kTcTicks = 128, kTcThreads = 256;
__device__ int g_tc_error;                                   // a wait on the tensor cores ran out (fg_mem_sync)

__device__ __forceinline__ bool tc_wait_one(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!fg::mbar_try(bar, parity))
        if (clock64() - t0 > fg::kTcWaitCycles) {
            atomicExch(&g_tc_error, 1);
            return false;
        }
    return true;
}
// the same by a whole warp, which stays together
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity) {
    const bool ok = tc_wait_one(bar, parity);
    return __all_sync(0xffffffffu, ok);
}
// what a thread loaded from TMEM may be used after this
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_bf16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
// instruction descriptor: fp32 accumulator, A and B bf16, M = 128; the operands' forms (0 K-major, 1 MN-major)
__device__ __forceinline__ uint32_t bf16_idesc(uint32_t n, uint32_t a_mn, uint32_t b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void async_copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// (x, y) as two bf16 pairs: the rounded values and what is left of them
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack_bf16(x, y);
    lo = pack_bf16(x - bf16_lo(hi), y - bf16_hi(hi));
}

struct TcLayout {
    uint32_t a, b, c, stage, state, table, bars, bytes;
};
__host__ __device__ inline TcLayout tc_layout(int D, int E) {
    TcLayout l;
    l.a = 0;
    l.b = kTcTicks * D * 2;
    l.c = 2 * l.b;
    l.stage = l.c + kTcTicks * E * 2;
    l.state = 2 * l.stage;
    l.table = l.state + D * E * 2;
    l.bars = l.table + 132 * 4;
    l.bytes = l.bars + 64;
    if (D < 128) l.bytes += 2048;      // an M = 128 operand of fewer rows reads past its own last core matrices
    return l;
}

// WIDE (dim or value_dim over 64): one block a SM, all 512 TMEM columns; else two, 256 columns each, dS in A's place.
template <bool BACK, bool WIDE>
__global__ void __launch_bounds__(kTcThreads, WIDE ? 1 : 2) k_decay_tc(const __grid_constant__ Scan s, int parts_only) {
    extern __shared__ __align__(1024) unsigned char smem[];
    constexpr int kBlocks = WIDE ? 4 : 2;                     // a thread's 16-column blocks of a state row
    const TcLayout lay = tc_layout(s.D, s.E);
    float* pw = reinterpret_cast<float*>(smem + lay.table);   // gamma^0 .. gamma^128
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + lay.bars);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4);
    const uint32_t sm = fg::smem_u32(smem), bar0 = fg::smem_u32(bars);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;   // the thread's TMEM lane = tick of A, O; row of S
    const int D = s.D, E = s.E, CD = D / 8, CE = E / 8, NE = E / 16;
    const int h = blockIdx.x % s.heads, part = blockIdx.y;
    const long long b = blockIdx.x / s.heads;
    const Span sp = span_of(s, b);
    const long long per = part_ticks(sp.n, s.parts), t0 = min(sp.n, part * per), t1 = min(sp.n, t0 + per);
    const bool hand_on = !parts_only && s.last && (sp.n ? t1 == sp.n && t1 > t0 : part == 0);
    if (t1 == t0 && !hand_on && !parts_only) return;
    const float ld = s.log_decay[h];

    if (tid == 0)
        for (int i = 0; i < 4; ++i) fg::mbar_init(bar0 + 8 * i, 1);
    if (tid == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fg::smem_u32(tmem_slot)),
                     "r"(WIDE ? 512 : 256)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (int i = tid; i <= kTcTicks; i += kTcThreads) pw[i] = power(ld, (float)i);

    // tick r of the chunk that starts t ticks into the scan (n ticks): the recording's tick, rows in recording order
    auto tick_of = [&](long long t, int n) { return sp.start + (BACK ? sp.n - t - n : t); };
    auto load = [&](const Operand& o, uint32_t at, int C, long long first, int n) {
        const char* p = o.p + 2 * ((s.offsets ? 0 : b * o.batch) + first * o.tick + (h / o.share) * o.head);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int rg = warp + 8 * g, r = rg * 8 + (lane & 7);
            const char* q = p + 2 * (r < n ? (long long)r * o.tick : 0);
            const uint32_t dst = at + (uint32_t)(rg * C) * 128 + (lane & 7) * 16;
            for (int c = lane >> 3; c < C; c += 4) async_copy16(dst + c * 128, q + c * 16, r < n);
        }
    };
    auto load_chunk = [&](long long t, uint32_t stage) {
        const int n = (int)min((long long)kTcTicks, t1 - t);
        const long long first = tick_of(t, n);
        if (!parts_only) load(s.a, stage + lay.a, CD, first, n);
        load(s.b, stage + lay.b, CD, first, n);
        load(s.c, stage + lay.c, CE, first, n);
    };
    if (t1 > t0) load_chunk(t0, sm);
    asm volatile("cp.async.commit_group;" ::: "memory");

    // the state before this part
    float S[kBlocks][16];
    const long long state0 = (b * s.heads + h) * D * E;
    const bool mine = row < D;
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
        const int e0 = (2 * j + half) * 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) S[j][i] = 0.f;
        if (parts_only || !mine || e0 >= E) continue;
        if (s.first) {
            const float f = power(ld, (float)(BACK ? max(t0 - 1, 0ll) : t0));
#pragma unroll
            for (int i = 0; i < 16; ++i)
                S[j][i] = f * s.first[state0 + (s.first_t ? (long long)(e0 + i) * D + row : (long long)row * E + e0 + i)];
        }
        for (int p = 0; p < part; ++p) {
            const float f = power(ld, (float)(t0 - min(sp.n, (p + 1) * per)));
            const float4* q = reinterpret_cast<const float4*>(
                s.partial + ((b * s.heads + h) * s.parts + p) * D * E + (long long)row * E + e0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 v = q[i];
                S[j][4 * i] = fmaf(f, v.x, S[j][4 * i]);
                S[j][4 * i + 1] = fmaf(f, v.y, S[j][4 * i + 1]);
                S[j][4 * i + 2] = fmaf(f, v.z, S[j][4 * i + 2]);
                S[j][4 * i + 3] = fmaf(f, v.w, S[j][4 * i + 3]);
            }
        }
    }
    auto put_state = [&]() {                                 // S as the operand of O1: rows d, columns e
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
            const int blk = 2 * j + half;
            if (!mine || blk >= NE) continue;
            uint4* at = reinterpret_cast<uint4*>(smem + lay.state + ((row >> 3) * CE + blk * 2) * 128 + (row & 7) * 16);
            at[0] = make_uint4(pack_bf16(S[j][0], S[j][1]), pack_bf16(S[j][2], S[j][3]), pack_bf16(S[j][4], S[j][5]),
                               pack_bf16(S[j][6], S[j][7]));
            at[8] = make_uint4(pack_bf16(S[j][8], S[j][9]), pack_bf16(S[j][10], S[j][11]), pack_bf16(S[j][12], S[j][13]),
                               pack_bf16(S[j][14], S[j][15]));
        }
    };
    if (!parts_only) put_state();
    fg::tc_fence_before();
    __syncthreads();
    fg::tc_fence_after();
    const uint32_t tmem = *tmem_slot, lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tA = 0, tO1 = 128, tO2 = tO1 + (WIDE ? 128 : 64), tS = WIDE ? 384 : 0;
    bool ok = true;
    int lead = BACK && s.first && part == 0 && !parts_only ? 0 : 1;    // exponent of S at the chunk's first tick

    for (long long t = t0; t < t1; t += kTcTicks) {
        const int it = (int)((t - t0) / kTcTicks), n = (int)min((long long)kTcTicks, t1 - t);
        const uint32_t stage = sm + (it & 1) * lay.stage, parity = it & 1;
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (tid == 0 && !parts_only) {
            fg::tc_fence_after();
            for (int k = 0; k < D / 16; ++k)
                mma_bf16(tmem + tA, fg::smem_desc(stage + lay.a + k * 256, 128, CD * 128),
                         fg::smem_desc(stage + lay.b + k * 256, 128, CD * 128), bf16_idesc(128, 0, 0), k > 0);
            fg::mma_commit(bar0);
            for (int k = 0; k < D / 16; ++k)
                mma_bf16(tmem + tO1, fg::smem_desc(stage + lay.a + k * 256, 128, CD * 128),
                         fg::smem_desc(sm + lay.state + k * 2 * CE * 128, CE * 128, 128), bf16_idesc(E, 0, 1), k > 0);
            fg::mma_commit(bar0 + 8);
        }
        __syncwarp();
        if (t + kTcTicks < t1) load_chunk(t + kTcTicks, sm + ((it + 1) & 1) * lay.stage);
        asm volatile("cp.async.commit_group;" ::: "memory");

        uint32_t hi[4][8], lo[4][8];
        if (!parts_only) {
            if (ok) ok = tc_wait(bar0, parity);
            fg::tc_fence_after();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int s0 = (2 * j + half) * 16, w0 = (warp & 3) * 32;
                // a block of 16 columns that no row of the warp reaches is 0; one that every row reaches in full takes
                // gamma^{t-s} as two factors <= 1; a block on the diagonal looks each weight up
                if (BACK ? s0 + 15 < w0 : s0 > w0 + 31) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) hi[j][i] = lo[j][i] = 0;
                    continue;
                }
                uint32_t v[16];
                fg::tmem_ld16(lanes + tA + s0, v);
                tmem_ready(v);
                if (BACK ? s0 >= w0 + 31 : s0 + 15 <= w0) {
                    const float f = pw[BACK ? s0 - row : row - s0 - 15];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float g0 = pw[BACK ? 2 * i : 15 - 2 * i], g1 = pw[BACK ? 2 * i + 1 : 14 - 2 * i];
                        split2(__uint_as_float(v[2 * i]) * (f * g0), __uint_as_float(v[2 * i + 1]) * (f * g1), hi[j][i], lo[j][i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d0 = BACK ? s0 + 2 * i - row : row - s0 - 2 * i, d1 = BACK ? d0 + 1 : d0 - 1;
                        const float x = d0 >= 0 ? __uint_as_float(v[2 * i]) * pw[d0] : 0.f;
                        const float y = d1 >= 0 ? __uint_as_float(v[2 * i + 1]) * pw[d1] : 0.f;
                        split2(x, y, hi[j][i], lo[j][i]);
                    }
                }
            }
            if (ok) ok = tc_wait(bar0 + 8, parity);            // O1 is done with a
        }
        // b' = gamma^{n-1-r} b in two terms, over b and a
        unsigned char* st = smem + (it & 1) * lay.stage;
        for (int u = tid; u < kTcTicks * CD; u += kTcThreads) {
            const int r = (u >> 3) / CD * 8 + (u & 7);
            const float f = pw[BACK ? r : max(n - 1 - r, 0)];
            uint4 v = *reinterpret_cast<uint4*>(st + lay.b + u * 16), l;
            split2(bf16_lo(v.x) * f, bf16_hi(v.x) * f, v.x, l.x);
            split2(bf16_lo(v.y) * f, bf16_hi(v.y) * f, v.y, l.y);
            split2(bf16_lo(v.z) * f, bf16_hi(v.z) * f, v.z, l.z);
            split2(bf16_lo(v.w) * f, bf16_hi(v.w) * f, v.w, l.w);
            *reinterpret_cast<uint4*>(st + lay.b + u * 16) = v;
            *reinterpret_cast<uint4*>(st + lay.a + u * 16) = l;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fg::tc_fence_before();
        if (!__syncthreads_and(ok)) break;                    // every thread has read A; b' is in place
        fg::tc_fence_after();
        auto issue_state = [&]() {
            const uint32_t id = bf16_idesc(E, 1, 1);
            for (int term = 0; term < 2; ++term)
                for (int k = 0; k < kTcTicks / 16; ++k)
                    mma_bf16(tmem + tS, fg::smem_desc(stage + (term ? lay.a : lay.b) + k * 2 * CD * 128, CD * 128, 128),
                             fg::smem_desc(stage + lay.c + k * 2 * CE * 128, CE * 128, 128), id, term + k > 0);
            fg::mma_commit(bar0 + 24);
        };
        if ((WIDE || parts_only) && tid == 0) issue_state();
        __syncwarp();
        if (!parts_only) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                tmem_st8(lanes + tA + (2 * j + half) * 8, hi[j]);
                tmem_st8(lanes + tA + 64 + (2 * j + half) * 8, lo[j]);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fg::tc_fence_before();
            __syncthreads();
            if (tid == 0) {
                fg::tc_fence_after();
                const uint32_t id = bf16_idesc(E, 0, 1);
                for (int term = 0; term < 2; ++term)
                    for (int k = 0; k < kTcTicks / 16; ++k)
                        mma_bf16_tmem(tmem + tO2, tmem + tA + term * 64 + k * 8,
                                      fg::smem_desc(stage + lay.c + k * 2 * CE * 128, CE * 128, 128), id, term + k > 0);
                fg::mma_commit(bar0 + 16);
                if (!WIDE) {
                    ok = tc_wait_one(bar0 + 16, parity) && ok;    // dS takes A's columns
                    issue_state();
                }
            }
        }
        // S, in registers, and as the next chunk's operand
        ok = __all_sync(0xffffffffu, ok);
        ok = tc_wait(bar0 + 24, parity) && ok;
        fg::tc_fence_after();
        const float fade = pw[n - 1 + lead];
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
            if (2 * j + half >= NE) continue;
            uint32_t v[16];
            fg::tmem_ld16(lanes + tS + (2 * j + half) * 16, v);
            tmem_ready(v);
#pragma unroll
            for (int i = 0; i < 16; ++i) S[j][i] = fmaf(S[j][i], fade, s.scale_in * __uint_as_float(v[i]));
        }
        if (!parts_only) {
            put_state();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            ok = tc_wait(bar0 + 16, parity) && ok;
            fg::tc_fence_after();
            const float f = pw[max(BACK ? n - 1 - row : row, 0) + lead] * s.scale_out;
            const long long first = tick_of(t, n);
            const long long at = (s.offsets ? 0 : b * s.out.batch) + (first + row) * s.out.tick + h * s.out.head;
#pragma unroll
            for (int j = 0; j < kBlocks; ++j) {
                const int e0 = (2 * j + half) * 16;
                if (e0 >= E) continue;
                __syncwarp();
                uint32_t x[16], y[16];
                fg::tmem_ld16(lanes + tO1 + e0, x);
                fg::tmem_ld16(lanes + tO2 + e0, y);
                tmem_ready(x);
                tmem_ready(y);
                float o[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = fmaf(__uint_as_float(x[i]), f, __uint_as_float(y[i]) * (s.scale_in * s.scale_out));
                if (row >= n) continue;
                if (s.out_f32) {
                    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(s.out.p) + at + e0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else {
                    uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(s.out.p) + at + e0);
                    p[0] = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
                    p[1] = make_uint4(pack_bf16(o[8], o[9]), pack_bf16(o[10], o[11]), pack_bf16(o[12], o[13]), pack_bf16(o[14], o[15]));
                }
            }
        }
        lead = 1;
        fg::tc_fence_before();                                // (the loop's first barrier orders these reads)
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    ok = __syncthreads_and(ok);
    if (!ok) {                                                // say so in what is handed on, too
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) S[j][i] = __int_as_float(0x7fc00000);
    }
    float* to = parts_only ? s.partial + ((b * s.heads + h) * s.parts + part) * D * E : hand_on ? s.last + state0 : nullptr;
    if (to && mine) {
        const bool across = !parts_only && s.last_t;
        const float f = !parts_only && BACK && sp.n ? pw[1] : 1.f;
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
            const int e0 = (2 * j + half) * 16;
            if (e0 >= E) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i) to[across ? (long long)(e0 + i) * D + row : (long long)row * E + e0 + i] = f * S[j][i];
        }
    }
    fg::tc_fence_after();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(WIDE ? 512 : 256) : "memory");
}

inline bool whole_units(const Operand& o) {                  // 16-byte copies fit
    return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.batch % 8 == 0 && o.tick % 8 == 0 && o.head % 8 == 0;
}
inline bool tc_fits(const Scan& s) {
    return s.D % 16 == 0 && s.E % 16 == 0 && s.D <= 128 && s.E <= 128 && whole_units(s.a) && whole_units(s.b) &&
           whole_units(s.c) && whole_units(s.out);
}
template <bool BACK, bool WIDE>
void tc_launch_as(const Scan& s, cudaStream_t st) {
    const TcLayout l = tc_layout(s.D, s.E);
    MCK(cudaFuncSetAttribute(k_decay_tc<BACK, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)l.bytes));
    const unsigned rows = (unsigned)(s.batch * s.heads);
    if (s.parts > 1) k_decay_tc<BACK, WIDE><<<dim3(rows, s.parts - 1), kTcThreads, l.bytes, st>>>(s, 1);
    k_decay_tc<BACK, WIDE><<<dim3(rows, s.parts), kTcThreads, l.bytes, st>>>(s, 0);
    MCK(cudaGetLastError());
}
inline void tc_launch(const Scan& s, cudaStream_t st) {
    const bool wide = s.D > 64 || s.E > 64;
    if (s.backward) wide ? tc_launch_as<true, true>(s, st) : tc_launch_as<true, false>(s, st);
    else wide ? tc_launch_as<false, true>(s, st) : tc_launch_as<false, false>(s, st);
}

}  // namespace
