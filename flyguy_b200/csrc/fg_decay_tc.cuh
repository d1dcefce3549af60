// The decay scan of bf16 operands on the tensor cores (tcgen05 kind::f16, accumulators in TMEM), chunks of 128 ticks:
//
//   out_t = scale_out (gamma^{t+1} a_t S + scale_in sum_{s<=t} gamma^{t-s} (a_t b_s) c_s)     t, s: ticks of the chunk
//   S    <- gamma^n S + scale_in sum_s gamma^{n-1-s} b_s c_s^T                                n: ticks of the chunk
//
// (run from the back: s >= t, gamma^{s-t}, exponents mirrored). Four products a chunk:
//   A  [128 x 128] = a b^T                operands as they arrive, exact products
//   O1 [128 x E]   = a S                  S rounded to bf16
//   O2 [128 x E]   = W c                  W = A . gamma^{t-s} as two bf16 terms (2^-17), over A in TMEM
//   dS [D x E]     = b'^T c               b' = gamma^{n-1-s} b as three bf16 terms (2^-25), over b, a and the copy of S
// S itself stays in fp32 registers for the whole recording, thread = row, so states are as good as fp32 sums. The one
// rounding to bf16, of S in O1, is of the size of the rounding of out itself.
//
// Tiles lie in shared memory as TMA writes them, 64 values (128 bytes, swizzled) of a tick in a row: read along the values
// or along the ticks that is the K-major or the MN-major form of the same bytes, so nothing is transposed.
//
// 20 warps: 0-7 the ticks (A to W, O1 and O2 to out; warps w and w + 4 share TMEM lanes 32 (w % 4) .. and take alternate
// blocks of 32 columns), 8-15 the state (b to b', S), 16 the copies and the MMAs. The roles meet at mbarriers only, so a
// chunk's elementwise work runs beside its MMAs and the next chunk's copies.
#pragma once
#include <cuda.h>

#include "fg_memory.cuh"
#include "fg_tcgen05.cuh"

namespace {
using namespace fgm;

constexpr int kTcTicks = 128, kTcThreads = 20 * 32;
__device__ int g_tc_error;                                   // a wait ran out (fg_mem_sync)

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
// 128-byte swizzle; rows of 128 bytes, 8 of them 1,024 bytes. K-major: `next` is unused; MN-major: from one 64 values to
// the next.
__device__ __forceinline__ uint64_t swizzled(uint32_t addr, uint32_t next) {
    return fg::smem_desc(addr, next, 1024) | (2ull << 61);
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) { fg::tmem_ld16(addr, r); }
// what a thread loaded from TMEM may be used after this
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// (x, y) rounded to a bf16 pair, and what is left of them
__device__ __forceinline__ uint32_t take_bf16(float& x, float& y) {
    const uint32_t r = pack_bf16(x, y);
    x -= bf16_lo(r);
    y -= bf16_hi(r);
    return r;
}
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int x, int head, int tick, int batch,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(tick), "r"(batch), "r"(bar)
        : "memory");
}

// Bounded wait for a barrier's phase. A try suspends the thread until the phase or about 0.1 ms are over, so that waiting
// warps leave shared memory to the MMAs' operands.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    const long long t0 = clock64();
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 100000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (*gave_up) return false;
        if (clock64() - t0 > fg::kTcWaitCycles) {
            *gave_up = 1;
            atomicExch(&g_tc_error, 1);
            return false;
        }
    }
}

__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int x, int head, int tick, int batch) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map),
                 "r"(x), "r"(head), "r"(tick), "r"(batch), "r"(src)
                 : "memory");
}
// the stores that this thread has issued have left shared memory
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

struct TcMaps {
    CUtensorMap a, b, c, out;
};
// DP, EP: dim and value_dim up to 64 or 128
template <int DP, int EP>
struct TcLayout {
    static constexpr uint32_t a = 0, b = kTcTicks * DP * 2, c = 2 * b, stage = c + kTcTicks * EP * 2;
    static constexpr uint32_t state = 2 * stage;             // the copy of S, then the third term of b'
    static constexpr uint32_t after = state + (DP * EP * 2 > kTcTicks * DP * 2 ? DP * EP * 2 : kTcTicks * DP * 2);
    // where a chunk of out is put together: room for fp32, or (no room left) where its c was, fp32 in two halves
    static constexpr bool own_out = DP + EP < 256;
    static constexpr uint32_t table = after + (own_out ? kTcTicks * EP * 4 : 0);
    static constexpr uint32_t bars = table + (32 + 132 + 16) * 4;
    static constexpr uint32_t bytes = bars + 128;
};
enum { kFull0, kFull1, kQk, kQs, kPv, kKv, kCFree, kWReady, kBReady, kSReady, kOutRead, kMeet, kBars };

// PARTS: the states of the parts alone
template <int DP, int EP, bool BACK, bool PARTS>
__global__ void __launch_bounds__(kTcThreads, 1) k_decay_tc(const __grid_constant__ Scan s,
                                                            const __grid_constant__ TcMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using L = TcLayout<DP, EP>;
    constexpr uint32_t kBox = kTcTicks * 128, kStateBox = DP * 128;
    constexpr int kTmem = 512;
    constexpr uint32_t tA = 0, tO1 = 128, tO2 = tO1 + EP, tS = tO2 + EP;
    float* pw = reinterpret_cast<float*>(smem + L::table) + 32;   // gamma^0 .. gamma^128, before them zeros
    float* ramp = pw + 132;                                  // gamma^{15-j}, from the back gamma^j
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t sm = fg::smem_u32(smem), bar0 = fg::smem_u32(bars);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = s.D, E = s.E;
    const int h = blockIdx.x % s.heads, part = blockIdx.y;
    const long long b = blockIdx.x / s.heads;
    const Span sp = span_of(s, b);
    const long long per = part_ticks(sp.n, s.parts), t0 = min(sp.n, part * per), t1 = min(sp.n, t0 + per);
    const bool hand_on = !PARTS && s.last && (sp.n ? t1 == sp.n && t1 > t0 : part == 0);
    if (t1 == t0 && !hand_on && !PARTS) return;
    const int chunks = (int)((t1 - t0 + kTcTicks - 1) / kTcTicks);
    const float ld = s.log_decay[h];

    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    if (tid == 0) {
        for (int i = 0; i < kBars; ++i) fg::mbar_init(bar(i), i >= kWReady ? 8 : 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fg::smem_u32(tmem_slot)),
                     "r"(kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (int i = tid; i <= kTcTicks; i += kTcThreads) pw[i] = power(ld, (float)i);
    if (tid < 32) pw[-1 - tid] = 0.f;
    if (tid < 16) ramp[tid] = power(ld, (float)(BACK ? tid : 15 - tid));
    fg::tc_fence_before();
    __syncthreads();
    fg::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // chunk i: its ticks, and the recording's tick of its first row (rows in recording order)
    auto ticks_of = [&](int i) { return (int)min((long long)kTcTicks, t1 - t0 - (long long)i * kTcTicks); };
    auto first_of = [&](int i) {
        const long long t = t0 + (long long)i * kTcTicks;
        return sp.start + (BACK ? sp.n - t - ticks_of(i) : t);
    };
    auto wait = [&](int i, int chunk) { return tc_wait(bar(i), (uint32_t)chunk & 1, gave_up); };
    auto wait_warp = [&](int i, int chunk) {
        const bool ok = wait(i, chunk);
        const bool all = __all_sync(0xffffffffu, ok);
        fg::tc_fence_after();
        return all;
    };
    auto arrive = [&](int i) {                               // a warp's threads are all done
        __syncwarp();
        if (lane == 0) fg::mbar_arrive(bar(i));
    };
    // with `first`, run from the back, S counts undecayed at the first tick
    const int lead0 = BACK && s.first && part == 0 && !PARTS ? 0 : 1;
    bool ok = true;

    // 20 warps start with 96 registers a thread: 640 x 96 = 61,440. The copies and MMAs (and the three warps beside them, there
    // because registers change hands by four warps) keep 48, the ticks 88, so that the state has 128 (S alone is 64):
    // 128 x 48 + 256 x 88 + 256 x 128 = 61,440
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        // ---- copies and MMAs -----------------------------------------------------------------------------------
        if (warp == 16 && lane == 0) {
            const int da = (D + 63) / 64, ec = (E + 63) / 64, batch = s.offsets ? 0 : (int)b;
            auto copy = [&](int i) {                         // a and b (and the bytes that c will add)
                const uint32_t stage = sm + (i & 1) * L::stage, full = bar(kFull0 + (i & 1));
                const int tick = (int)first_of(i);
                fg::mbar_expect_tx(full, (uint32_t)((PARTS ? 1 : 2) * da + ec) * kBox);
                for (int x = 0; x < da; ++x) {
                    if (!PARTS) tma_tile(stage + L::a + x * kBox, &maps.a, x * 64, h / s.a.share, tick, batch, full);
                    tma_tile(stage + L::b + x * kBox, &maps.b, x * 64, h / s.b.share, tick, batch, full);
                }
            };
            auto copy_c = [&](int i) {
                const uint32_t stage = sm + (i & 1) * L::stage, full = bar(kFull0 + (i & 1));
                for (int x = 0; x < ec; ++x)
                    tma_tile(stage + L::c + x * kBox, &maps.c, x * 64, h / s.c.share, (int)first_of(i), batch, full);
            };
            // 16 values of a K-major tile; 16 ticks (rows) of an MN-major one; descriptors count in 16 bytes
            constexpr auto along = [](int k) { return (uint64_t)((k >> 2) * kBox + (k & 3) * 32) >> 4; };
            constexpr auto down = [](int k) { return (uint64_t)(k * 2048) >> 4; };
            const uint32_t id_a = bf16_idesc(128, 0, 0), id_o = bf16_idesc(E, 0, 1), id_s = bf16_idesc(E, 1, 1);
            const uint64_t state_rows = swizzled(sm + L::state, kStateBox);
            constexpr uint32_t next_b = DP == 128 ? kBox : 0;     // (an M = 128 operand of 64 values: twice the same)
            int started = 0, copied = 0;                     // chunks whose a and b, and whose c too, are on their way
            if (chunks) { copy(0); copy_c(0); started = copied = 1; }
            for (int i = 0; i < chunks && ok; ++i) {
                const uint32_t stage = sm + (i & 1) * L::stage;
                const uint64_t a_ticks = swizzled(stage + L::a, 0), b_ticks = swizzled(stage + L::b, 0),
                               c_rows = swizzled(stage + L::c, kBox);
                const uint64_t terms[3] = {swizzled(stage + L::b, next_b), swizzled(stage + L::a, next_b), swizzled(sm + L::state, next_b)};
                if (i > 0) ok = wait(kKv, i - 1) && (PARTS || wait(kPv, i - 1));   // the other stage is free, and A
                if (!ok) break;
                const bool more = i + 1 < chunks, wait_c = !PARTS && !L::own_out && i > 0;
                if (more) { copy(i + 1); ++started; }
                if (more && !wait_c) { copy_c(i + 1); ++copied; }
                ok = tc_wait(bar(kFull0 + (i & 1)), (i >> 1) & 1, gave_up);
                if (!ok) break;
                fg::tc_fence_after();
                if (!PARTS) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_bf16(tmem + tA, a_ticks + along(k), b_ticks + along(k), id_a, k > 0);
                    fg::mma_commit(bar(kQk));
                    if (more && wait_c) {                    // out of the chunk before has left c's place
                        ok = wait(kCFree, i - 1);
                        if (!ok) break;
                        copy_c(i + 1);
                        ++copied;
                    }
                    ok = wait(kSReady, i) && (i == 0 || wait(kOutRead, i - 1));
                    if (!ok) break;
                    fg::tc_fence_after();
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_bf16(tmem + tO1, a_ticks + along(k), state_rows + down(k), id_o, k > 0);
                    fg::mma_commit(bar(kQs));
                    ok = wait(kWReady, i) && (ticks_of(i) == kTcTicks || wait(kBReady, i));   // (c's end is cleared there)
                    if (!ok) break;
                    fg::tc_fence_after();
#pragma unroll
                    for (int term = 0; term < 2; ++term)
#pragma unroll
                        for (int k = 0; k < kTcTicks / 16; ++k)
                            mma_bf16_tmem(tmem + tO2, tmem + tA + k * 16 + term * 8, c_rows + down(k), id_o, term + k > 0);
                    fg::mma_commit(bar(kPv));
                } else {
                    fg::mma_commit(bar(kQk));                // (nothing before it: the tile has arrived)
                    ok = wait(kSReady, i);                   // dS has been read
                    if (!ok) break;
                }
                ok = wait(kBReady, i);
                if (!ok) break;
                fg::tc_fence_after();
#pragma unroll
                for (int term = 0; term < 3; ++term)
#pragma unroll
                    for (int k = 0; k < kTcTicks / 16; ++k)
                        mma_bf16(tmem + tS, terms[term] + down(k), c_rows + down(k), id_s, term + k > 0);
                fg::mma_commit(bar(kKv));
            }
            if (!ok && copied < started) copy_c(copied++);
            if (!ok)                                         // let the copies in flight land before the block ends
                for (int i = max(0, copied - 2); i < copied; ++i) {
                    const long long c0 = clock64();
                    while (!fg::mbar_try(bar(kFull0 + (i & 1)), (i >> 1) & 1) && clock64() - c0 < fg::kTcWaitCycles) {}
                }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // ---- ticks ---------------------------------------------------------------------------------------------
        const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        int meetings = 0;
        auto meet = [&]() {                                  // the eight warps wait for one another
            arrive(kMeet);
            return wait_warp(kMeet, meetings++);
        };
        for (int i = 0; !PARTS && i < chunks && ok; ++i) {
            const int n = ticks_of(i);
            ok = wait_warp(kQk, i);
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int blk = 2 * j + half;                 // blocks of 32 on one side of the diagonal are 0
                uint32_t v[2][16], hi[8], lo[8];
                if (BACK ? blk < quarter : blk > quarter) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) hi[k] = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) tmem_st8(lanes + tA + blk * 32 + k * 8, hi);
                    continue;
                }
                tmem_ld16(lanes + tA + blk * 32, v[0]);
                tmem_ld16(lanes + tA + blk * 32 + 16, v[1]);
                tmem_ready(v[0]);
                tmem_ready(v[1]);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int s0 = blk * 32 + q * 16;
                    if (BACK && n < kTcTicks) {               // the last ticks are not the chunk's
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (s0 + k >= n) v[q][k] = 0;
                    }
                    if (blk != quarter) {                    // gamma^{t-s} as two factors, both at most 1
                        const float f = pw[BACK ? s0 - row : row - s0 - 15];
                        const float4* r4 = reinterpret_cast<const float4*>(ramp);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float4 g = r4[k];
                            float x0 = __uint_as_float(v[q][4 * k]) * (f * g.x), x1 = __uint_as_float(v[q][4 * k + 1]) * (f * g.y);
                            float x2 = __uint_as_float(v[q][4 * k + 2]) * (f * g.z), x3 = __uint_as_float(v[q][4 * k + 3]) * (f * g.w);
                            hi[2 * k] = take_bf16(x0, x1);
                            lo[2 * k] = pack_bf16(x0, x1);
                            hi[2 * k + 1] = take_bf16(x2, x3);
                            lo[2 * k + 1] = pack_bf16(x2, x3);
                        }
                    } else {
                        const float* g = pw + (BACK ? s0 - row : row - s0);   // gamma^{t-s} in turn; 0 past the diagonal
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float x = __uint_as_float(v[q][2 * k]) * g[BACK ? 2 * k : -2 * k];
                            float y = __uint_as_float(v[q][2 * k + 1]) * g[BACK ? 2 * k + 1 : -2 * k - 1];
                            hi[k] = take_bf16(x, y);
                            lo[k] = pack_bf16(x, y);
                        }
                    }
                    tmem_st8(lanes + tA + s0, hi);
                    tmem_st8(lanes + tA + s0 + 8, lo);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fg::tc_fence_before();
            arrive(kWReady);
            const float f = pw[max(BACK ? n - 1 - row : row, 0) + (i ? 1 : lead0)] * s.scale_out;
            const float g = s.scale_in * s.scale_out;
            ok = wait_warp(kQs, i) && wait_warp(kPv, i);
            if (!ok) break;
            auto out16 = [&](int e0, float (&o)[16]) {
                uint32_t x[16], y[16];
                tmem_ld16(lanes + tO1 + e0, x);
                tmem_ld16(lanes + tO2 + e0, y);
                tmem_ready(x);
                tmem_ready(y);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = fmaf(__uint_as_float(x[k]), f, __uint_as_float(y[k]) * g);
            };
            if (n == kTcTicks) {
                // put together in shared memory, stored as one tile (a thread's own stores, 32 lines at a time, held up the
                // MMAs' operands: 4,000 instead of 1,900 clocks for dS)
                const uint32_t tile = L::own_out ? L::after : (i & 1) * L::stage + L::c;
                if (!L::own_out) {
                    ok = wait_warp(kKv, i);
                    if (!ok) break;
                }
                if (tid == 0) stores_read();
                ok = meet();
                if (!ok) break;
                const int halves = !L::own_out && s.out_f32 ? 2 : 1;
                for (int r = 0; r < halves && ok; ++r) {
#pragma unroll 1
                    for (int e0 = (halves == 2 ? r * 64 : 0) + half * 16; e0 < (halves == 2 ? min(E, r * 64 + 64) : E); e0 += 32) {
                        float o[16];
                        out16(e0, o);
                        const int x0 = halves == 2 ? e0 - r * 64 : e0;
                        if (s.out_f32) {
                            unsigned char* at = smem + tile + (x0 >> 5) * kBox + row * 128;
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                *reinterpret_cast<float4*>(at + (((((x0 & 31) >> 2) + k) ^ (row & 7)) << 4)) =
                                    make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                        } else {
                            unsigned char* at = smem + tile + (x0 >> 6) * kBox + row * 128;
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                *reinterpret_cast<uint4*>(at + (((((x0 & 63) >> 3) + k) ^ (row & 7)) << 4)) =
                                    make_uint4(pack_bf16(o[8 * k], o[8 * k + 1]), pack_bf16(o[8 * k + 2], o[8 * k + 3]),
                                               pack_bf16(o[8 * k + 4], o[8 * k + 5]), pack_bf16(o[8 * k + 6], o[8 * k + 7]));
                        }
                    }
                    if (r + 1 == halves) {
                        fg::tc_fence_before();
                        arrive(kOutRead);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    ok = meet();
                    if (ok && tid == 0) {
                        const int values = s.out_f32 ? 32 : 64, e1 = halves == 2 ? min(E, r * 64 + 64) : E;
                        for (int e0 = halves == 2 ? r * 64 : 0, x = 0; e0 < e1; e0 += values, ++x)
                            tma_store(&maps.out, sm + tile + x * kBox, e0, h, (int)first_of(i), s.offsets ? 0 : (int)b);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        if (!L::own_out) {
                            stores_read();
                            if (r + 1 == halves) fg::mbar_arrive(bar(kCFree));
                        }
                    }
                    __syncwarp();
                    if (r + 1 < halves) ok = ok && meet();
                }
            } else {                                          // a recording's last ticks: what follows them is another's
                const long long at = (s.offsets ? 0 : b * s.out.batch) + (first_of(i) + row) * s.out.tick + h * s.out.head;
#pragma unroll 1
                for (int e0 = half * 16; e0 < E; e0 += 32) {
                    float o[16];
                    out16(e0, o);
                    if (row < n && s.out_f32) {
                        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(s.out.p) + at + e0);
#pragma unroll
                        for (int k = 0; k < 4; ++k) p[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    } else if (row < n) {
                        uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(s.out.p) + at + e0);
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            p[k] = make_uint4(pack_bf16(o[8 * k], o[8 * k + 1]), pack_bf16(o[8 * k + 2], o[8 * k + 3]),
                                              pack_bf16(o[8 * k + 4], o[8 * k + 5]), pack_bf16(o[8 * k + 6], o[8 * k + 7]));
                    }
                    __syncwarp();
                }
                fg::tc_fence_before();
                arrive(kOutRead);
                if (!L::own_out && tid == 0) fg::mbar_arrive(bar(kCFree));
            }
        }
        if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        // ---- state ---------------------------------------------------------------------------------------------
        const int quarter = warp & 3, half = (warp >> 2) & 1, row = quarter * 32 + lane, st = tid - 256;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const bool mine = row < D;
        float S[EP / 32][16];
        const long long state0 = (b * s.heads + h) * D * E;
#pragma unroll
        for (int j = 0; j < EP / 32; ++j) {
            const int e0 = (2 * j + half) * 16;
#pragma unroll
            for (int i = 0; i < 16; ++i) S[j][i] = 0.f;
            if (PARTS || !mine || e0 >= E) continue;
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
        auto put_state = [&]() {                             // S as the operand of O1: rows d, columns e, swizzled
            if (!PARTS) {
#pragma unroll
                for (int j = 0; j < EP / 32; ++j) {
                    const int e0 = (2 * j + half) * 16, unit = (e0 & 63) >> 3;
                    if (row < DP && e0 < E) {                // (rows past D: zeros, for the k-steps of 16 up to DP)
                        unsigned char* at = smem + L::state + (e0 >> 6) * kStateBox + row * 128;
                        const float* x = S[j];
                        *reinterpret_cast<uint4*>(at + ((unit ^ (row & 7)) << 4)) =
                            make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
                        *reinterpret_cast<uint4*>(at + (((unit + 1) ^ (row & 7)) << 4)) = make_uint4(
                            pack_bf16(x[8], x[9]), pack_bf16(x[10], x[11]), pack_bf16(x[12], x[13]), pack_bf16(x[14], x[15]));
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            fg::tc_fence_before();
            arrive(kSReady);
        };
        put_state();
        for (int i = 0; i < chunks && ok; ++i) {
            const int n = ticks_of(i);
            unsigned char* stage = smem + (i & 1) * L::stage;
            ok = wait_warp(kQk, i) && (PARTS || wait_warp(kQs, i));
            // (the tile itself: TMA's writes are seen through its own barrier)
            ok = ok && __all_sync(0xffffffffu, tc_wait(bar(kFull0 + (i & 1)), (i >> 1) & 1, gave_up));
            if (!ok) break;
            // b' in three terms, over b, a and the copy of S; ticks past the chunk's end (another recording's) become 0 in
            // b' and c, whatever they hold
            for (int u = n * 8 + st; n < kTcTicks && u < kTcTicks * 8; u += 256) {
#pragma unroll
                for (int x = 0; x < EP / 64; ++x) *reinterpret_cast<uint4*>(stage + L::c + x * kBox + u * 16) = make_uint4(0, 0, 0, 0);
            }
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = pw[BACK ? (st >> 3) + 32 * k : max(n - 1 - (st >> 3) - 32 * k, 0)];
#pragma unroll 1
            for (int x = 0; x < DP / 64; ++x) {
                unsigned char* at = stage + L::b + x * kBox + st * 16;
                unsigned char* at_lo = smem + L::state + x * kBox + st * 16;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint4 v = *reinterpret_cast<uint4*>(at + k * 4096), m, l;
                    if ((st >> 3) + 32 * k >= n) v = make_uint4(0, 0, 0, 0);
                    uint32_t* pv = &v.x;
                    uint32_t* pm = &m.x;
                    uint32_t* pl = &l.x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float y = bf16_lo(pv[j]) * f[k], z = bf16_hi(pv[j]) * f[k];
                        pv[j] = take_bf16(y, z);
                        pm[j] = take_bf16(y, z);
                        pl[j] = pack_bf16(y, z);
                    }
                    *reinterpret_cast<uint4*>(at + k * 4096) = v;
                    *reinterpret_cast<uint4*>(at - L::b + L::a + k * 4096) = m;
                    *reinterpret_cast<uint4*>(at_lo + k * 4096) = l;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(kBReady);
            ok = wait_warp(kKv, i);
            if (!ok) break;
            const float fade = pw[n - 1 + (i ? 1 : lead0)];
#pragma unroll
            for (int j = 0; j < EP / 32; ++j) {
                if ((2 * j + half) * 16 >= E) continue;
                uint32_t v[16];
                tmem_ld16(lanes + tS + (2 * j + half) * 16, v);
                tmem_ready(v);
#pragma unroll
                for (int k = 0; k < 16; ++k) S[j][k] = fmaf(S[j][k], fade, s.scale_in * __uint_as_float(v[k]));
            }
            if (i + 1 < chunks) put_state();
        }
        if (*gave_up) {                                      // say so in what is handed on, too
#pragma unroll
            for (int j = 0; j < EP / 32; ++j)
#pragma unroll
                for (int k = 0; k < 16; ++k) S[j][k] = __int_as_float(0x7fc00000);
        }
        float* to = PARTS ? s.partial + ((b * s.heads + h) * s.parts + part) * D * E : hand_on ? s.last + state0 : nullptr;
        if (to && mine) {
            const float f = !PARTS && BACK && sp.n ? pw[1] : 1.f;
#pragma unroll
            for (int j = 0; j < EP / 32; ++j) {
                const int e0 = (2 * j + half) * 16;
                if (e0 >= E) continue;
                if (!PARTS && s.last_t) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) to[(long long)(e0 + k) * D + row] = f * S[j][k];
                } else {
                    float4* p = reinterpret_cast<float4*>(to + (long long)row * E + e0);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        p[k] = make_float4(f * S[j][4 * k], f * S[j][4 * k + 1], f * S[j][4 * k + 2], f * S[j][4 * k + 3]);
                }
            }
        }
    }
    fg::tc_fence_before();
    __syncthreads();
    fg::tc_fence_after();
    if (warp == 16)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
}

// what 16-byte copies and tensor maps take: strides of dimensions that there is more than one of
inline bool whole_units(const Scan& s, const Operand& o) {
    const auto fits = [&](long long st, long long n) { return n <= 1 || (st % 8 == 0 && st > 0 && st < (1ll << 36)); };
    return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && fits(o.batch, s.offsets ? 1 : s.batch) && fits(o.tick, s.ticks) &&
           fits(o.head, s.heads / o.share);
}
inline bool tc_fits(const Scan& s) {
    return s.D % 16 == 0 && s.E % 16 == 0 && s.D <= 128 && s.E <= 128 && s.ticks < (1ll << 31) && s.ticks > 0 &&
           s.batch < (1ll << 31) && whole_units(s, s.a) && whole_units(s, s.b) && whole_units(s, s.c) &&
           whole_units(s, s.out) && reinterpret_cast<uintptr_t>(s.last) % 16 == 0;
}
// [batch][ticks][heads][dim] as tiles of 128 bytes x 128 ticks, zeros outside
inline CUtensorMap tile_map(const Scan& s, const Operand& o, int dim, bool f32 = false) {
    const cuuint64_t size = f32 ? 4 : 2;
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        MCK(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q));
        need(f && q == cudaDriverEntryPointSuccess, "the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<Encode>(f);
    }();
    CUtensorMap m;
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)(s.heads / o.share), (cuuint64_t)s.ticks,
                                (cuuint64_t)(s.offsets ? 1 : s.batch)};
    const cuuint64_t st[3] = {dims[1] > 1 ? o.head * size : 16, dims[2] > 1 ? o.tick * size : 16,
                              dims[3] > 1 ? o.batch * size : 16};
    const cuuint32_t box[4] = {(cuuint32_t)(128 / size), 1, kTcTicks, 1}, step[4] = {1, 1, 1, 1};
    need(encode(&m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, o.p, dims, st, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
         "fg_decay_attn: no tensor map for these strides");
    return m;
}
template <int DP, int EP, bool BACK>
void tc_launch_as(const Scan& s, cudaStream_t st) {
    constexpr int bytes = TcLayout<DP, EP>::bytes;
    static const bool once = [] {
        MCK(cudaFuncSetAttribute(k_decay_tc<DP, EP, BACK, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        MCK(cudaFuncSetAttribute(k_decay_tc<DP, EP, BACK, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        return true;
    }();
    (void)once;
    const TcMaps maps{tile_map(s, s.a, s.D), tile_map(s, s.b, s.D), tile_map(s, s.c, s.E),
                      tile_map(s, s.out, s.E, s.out_f32)};
    const unsigned rows = (unsigned)(s.batch * s.heads);
    if (s.parts > 1) k_decay_tc<DP, EP, BACK, true><<<dim3(rows, s.parts - 1), kTcThreads, bytes, st>>>(s, maps);
    k_decay_tc<DP, EP, BACK, false><<<dim3(rows, s.parts), kTcThreads, bytes, st>>>(s, maps);
    MCK(cudaGetLastError());
}
template <bool BACK>
void tc_launch_dims(const Scan& s, cudaStream_t st) {
    if (s.D > 64) s.E > 64 ? tc_launch_as<128, 128, BACK>(s, st) : tc_launch_as<128, 64, BACK>(s, st);
    else s.E > 64 ? tc_launch_as<64, 128, BACK>(s, st) : tc_launch_as<64, 64, BACK>(s, st);
}
inline void tc_launch(const Scan& s, cudaStream_t st) {
    s.backward ? tc_launch_dims<true>(s, st) : tc_launch_dims<false>(s, st);
}

}  // namespace
