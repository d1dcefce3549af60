// The decay scan of bf16 operands on the tensor cores (tcgen05 kind::f16, accumulators in TMEM), chunks of 128 ticks:
//
//   out_t = scale_out (gamma^{t+1} a_t S + scale_in sum_{s<=t} gamma^{t-s} (a_t b_s) c_s)     t, s: ticks of the chunk
//   S    <- gamma^n S + scale_in sum_s gamma^{n-1-s} b_s c_s^T                                n: ticks of the chunk
//
// (run from the back: s >= t, gamma^{s-t}, exponents mirrored). Four products a chunk:
//   A  [128 x 128] = a b^T                operands as they arrive, exact products
//   O1 [128 x E]   = a S                  S rounded to bf16
//   O2 [128 x E]   = W c                  W = A . gamma^{t-s} rounded to bf16, over A in TMEM
//   dS [D x E]     = b'^T c               b' = gamma^{n-1-s} b as three bf16 terms (2^-25)
// S itself stays in fp32 registers for the whole recording, thread = row, so states are as good as fp32 sums. The roundings
// of S in O1 and of W in O2 are of the size of the rounding of out itself, and apart from one another: out is 2.3e-3 of its norm
// off where its own rounding alone is 1.7e-3. Second terms would take them away, but at 128 S's needs 32 KB more shared memory
// than there is (and W's alone leaves S's); callers are told. A tile is worked on at once, so a NaN or an infinity in c reaches
// all rows of its chunk (its weight for those before it is 0, and 0 times NaN is NaN), and an infinity in b' becomes a NaN.
//
// Tiles lie in shared memory as TMA writes them, 64 values (128 bytes, swizzled) of a tick in a row: read along the values
// or along the ticks that is the K-major or the MN-major form of the same bytes, so nothing is transposed. 227 KB hold two
// stages of a, b, c and a bf16 copy of S. At dim 64 the second and third terms of b' and out have places of their own; at
// 128 the terms go over a and the copy of S once O1 is done with both, and out (with a value_dim of 128, too) over c.
//
// 20 warps: 0-7 the ticks (A to W, O1 and O2 to out; warps w and w + 4 share TMEM lanes 32 (w % 4) .. and take alternate
// blocks of columns), 8-15 the state (S, b to b'), 16 and 18 the MMAs, 17 and 19 the copies in and
// out. The roles meet at mbarriers only, so a
// chunk's elementwise work runs beside its MMAs and the next chunk's copies.
//
// 64 recordings of 1,024 ticks, 8 heads of 128, forward: 189 us (403 MB in, 137 MB out; at the rate of a plain copy 82 us), 8
// chunks of 4.7 us a block and some 8 us around them, four rounds of blocks. What bounds it is the chain from one state to the
// next: S copied, O1, b' made (b is read and three terms written, 128 KB of shared memory at 128), 24 MMAs of dS (64 clocks
// each, for both operands come from shared memory), S read back. The tensor pipe is 26% busy, DRAM 35%, issue slots 31%. At dim
// 64 b' is made while O1 runs: 97,500 ticks, 8 heads, 190 us (250 MB). Blocks that took over one recording after another
// instead of ending (with the next one's first tiles on their way) lost more a chunk than they saved: forward and back took 2% longer.
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
__device__ __forceinline__ uint32_t pack2(uint64_t x) {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
    return pack_bf16(a, b);
}
__device__ __forceinline__ uint64_t unpack2(uint32_t v) { return two(bf16_lo(v), bf16_hi(v)); }
// a pair rounded to bf16, and what is left of it
__device__ __forceinline__ uint32_t take2(uint64_t& x) {
    const uint32_t r = pack2(x);
    x = fma2(unpack2(r), two(-1.f, -1.f), x);
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

// Bounded wait for a barrier's phase: a try suspends the thread until the phase or about 0.1 ms are over.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    for (int tries = 0;; ++tries) {
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
        if (tries > 20000) {                                 // (2 s)
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
    static constexpr bool own_terms = DP == 64, own_out = DP + EP < 256;
    static constexpr uint32_t a = 0, b = kTcTicks * DP * 2, c = 2 * b, stage = c + kTcTicks * EP * 2;
    static constexpr uint32_t state = 2 * stage;
    static constexpr uint32_t third = own_terms ? state + DP * EP * 2 : state, second = third + kTcTicks * DP * 2;   // (or over a)
    static constexpr uint32_t out = own_terms ? second + kTcTicks * DP * 2 : second, out_bytes = 32768;              // (or over c)
    static constexpr uint32_t table = out + (own_out ? out_bytes : 0);
    static constexpr uint32_t bars = table + (32 + 132) * 4;
    static constexpr uint32_t bytes = bars + 8 * 16 + 16;
    static_assert(own_terms || DP * EP * 2 <= kTcTicks * DP * 2, "the copy of S fits the third term's place");
};
// A wait tells odd phases from even ones only, so no phase may end before all that wait for the one before have seen it. kFull, kPv,
// kKv and kOutLeft are one barrier a stage: their next phase needs the copies into the stage, which come after those waits.
enum { kFull0, kFull1, kQk, kQs, kPv0, kPv1, kKv0, kKv1, kOutStored, kOutLeft0, kOutLeft1, kWReady, kBReady, kSReady, kOutRead, kOutReady, kBars };
static_assert(kBars <= 16, "room for the barriers");

// BACK: from the last tick to the first; F32: out in fp32; PARTS: the states of the parts alone
template <int DP, int EP, bool BACK, bool F32, bool PARTS>
__global__ void __launch_bounds__(kTcThreads, 1) k_decay_tc(const __grid_constant__ Scan s,
                                                            const __grid_constant__ TcMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using L = TcLayout<DP, EP>;
    constexpr uint32_t kBox = kTcTicks * 128, kStateBox = DP * 128;
    constexpr uint32_t tA = 0, tO1 = 128, tO2 = tO1 + EP, tS = tO2 + EP;
    float* pw = reinterpret_cast<float*>(smem + L::table) + 32;   // gamma^0 .. gamma^128, before them zeros
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t sm = fg::smem_u32(smem), bar0 = fg::smem_u32(bars);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = s.D, E = s.E;
    const int h = blockIdx.x % s.heads, part = blockIdx.y, b = blockIdx.x / s.heads;
    const bool last_block = s.beside && blockIdx.x == gridDim.x - 1;
    const Span sp = span_of(s, b);
    const long long per = part_ticks(sp.n, s.parts), t0 = min(sp.n, part * per), t1 = min(sp.n, t0 + per);
    const bool hand_on = !PARTS && s.last && (sp.n ? t1 == sp.n && t1 > t0 : part == 0);
    next_may_begin();
    if (t1 == t0 && !hand_on && !PARTS && !last_block) return;
    const int total = (int)(t1 - t0), chunks = (total + kTcTicks - 1) / kTcTicks;
    const float ld = s.log_decay[h];

    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    if (tid == 0) {
        for (int i = 0; i < kBars; ++i) fg::mbar_init(bar(i), i >= kWReady ? 8 : 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fg::smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid <= kTcTicks) pw[tid] = power(ld, (float)tid);
    else if (tid <= kTcTicks + 32) pw[kTcTicks - tid] = 0.f;
    fg::tc_fence_before();
    __syncthreads();
    fg::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // chunk i: its ticks, and the recording's tick of its first row (rows in recording order)
    const int begin = (int)(sp.start + (BACK ? sp.n - t0 : t0));
    auto ticks_of = [&](int i) { return min(kTcTicks, total - i * kTcTicks); };
    auto first_of = [&](int i) { return BACK ? begin - i * kTcTicks - ticks_of(i) : begin + i * kTcTicks; };
    const int batch = s.offsets ? 0 : b;
    auto wait = [&](int i, int chunk) { return tc_wait(bar(i), (uint32_t)chunk & 1, gave_up); };
    auto wait_stage = [&](int first, int chunk) { return tc_wait(bar(first + (chunk & 1)), (chunk >> 1) & 1, gave_up); };
    auto wait_full = [&](int i) { return wait_stage(kFull0, i); };
    auto together = [&](bool ok) {                           // a warp goes on, or not, as one
        ok = __all_sync(0xffffffffu, ok);
        fg::tc_fence_after();
        return ok;
    };
    auto arrive = [&](int i) {                               // a warp's threads are all done
        __syncwarp();
        if (lane == 0) fg::mbar_arrive(bar(i));
    };
    // b' = scale_in gamma^{..} b of chunk i (n ticks); ticks past its end (another recording's) become 0 in b' and c, whatever they hold.
    // Worker w of 256.
    auto fade_b = [&](int i, int n, int w) {
        constexpr int kWorkers = 256;
        unsigned char* stage = smem + (i & 1) * L::stage;
        unsigned char* second = L::own_terms ? smem + L::second : stage + L::a;
        if (n < kTcTicks)
            for (int u = n * 8 + w; u < kTcTicks * 8; u += kWorkers)
#pragma unroll
                for (int x = 0; x < EP / 64; ++x) *reinterpret_cast<uint4*>(stage + L::c + x * kBox + u * 16) = make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (int u = w; u < kTcTicks * DP / 8; u += kWorkers) {
            const int r = (u >> 3) & 127;
            const float f = pw[BACK ? r : max(n - 1 - r, 0)] * s.scale_in;
            uint4 v = *reinterpret_cast<uint4*>(stage + L::b + u * 16), m, l;
            if (r >= n) v = make_uint4(0, 0, 0, 0);
            uint32_t* pv = &v.x;
            uint32_t* pm = &m.x;
            uint32_t* pl = &l.x;
            const uint64_t f2 = two(f, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint64_t x = mul2(unpack2(pv[j]), f2);
                pv[j] = take2(x);
                pm[j] = take2(x);
                pl[j] = pack2(x);
            }
            *reinterpret_cast<uint4*>(stage + L::b + u * 16) = v;
            *reinterpret_cast<uint4*>(second + u * 16) = m;
            *reinterpret_cast<uint4*>(smem + L::third + u * 16) = l;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        arrive(kBReady);
    };
    // when b' may be made: b is no longer A's operand, the terms' places are free, and the tile has arrived (TMA's writes are
    // seen through its own barrier)
    auto b_free = [&](int i) {
        return (PARTS || wait(L::own_terms ? kQk : kQs, i)) && (i == 0 || wait_stage(kKv0, i - 1)) && wait_full(i);
    };
    // where a chunk of out is put together, and how many columns at a time
    auto out_at = [&](int i) { return L::own_out ? L::out : (i & 1) * L::stage + L::c; };
    constexpr int kRound = F32 ? 64 : 128;
    // with `first`, run from the back, S counts undecayed at the first tick
    const int lead0 = BACK && s.first && part == 0 && !PARTS ? 0 : 1;
    bool ok = true;

    // 20 warps start with 96 registers a thread: 640 x 96 = 61,440. The MMAs and copies keep 48, the ticks 88, so that the state has 128 (S alone is 64):
    // 128 x 48 + 256 x 88 + 256 x 128 = 61,440
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        // ---- copies and MMAs -----------------------------------------------------------------------------------
        if (warp == 17 && lane == 0) {
            // a chunk goes into the stage that the one before the last has left: its products are done, and its out, where it
            // is put together over c, is stored
            const int da = (D + 63) / 64, ec = (E + 63) / 64;
            const int head_a = h / s.a.share, head_b = h / s.b.share, head_c = h / s.c.share;
            int copied = 0;
#pragma unroll 1
            for (int i = 0; i < chunks && ok; ++i) {
                const uint32_t stage = sm + (i & 1) * L::stage, full = bar(kFull0 + (i & 1));
                const int tick = first_of(i);
                if (i >= 2)
                    ok = wait_stage(kKv0, i - 2) && (PARTS || (wait_stage(kPv0, i - 2) && (L::own_out || wait_stage(kOutLeft0, i - 2))));
                if (!ok) break;
                fg::mbar_expect_tx(full, (uint32_t)((PARTS ? 1 : 2) * da + ec) * kBox);
#pragma unroll 1
                for (int x = 0; x < da; ++x) {
                    if (!PARTS) tma_tile(stage + L::a + x * kBox, &maps.a, x * 64, head_a, tick, batch, full);
                    tma_tile(stage + L::b + x * kBox, &maps.b, x * 64, head_b, tick, batch, full);
                }
#pragma unroll 1
                for (int x = 0; x < ec; ++x) tma_tile(stage + L::c + x * kBox, &maps.c, x * 64, head_c, tick, batch, full);
                ++copied;
            }
            // (after a wait ran out, too) the copies land before the block ends
            for (int i = max(0, copied - 2); i < copied; ++i)
                for (int tries = 0; !fg::mbar_try(bar(kFull0 + (i & 1)), (i >> 1) & 1) && tries < 10000000; ++tries) {}
        } else if (warp == 16 && lane == 0 && !PARTS) {
            // A, O1 and O2. Unrolled: issued one by one in a loop they took longer than the tensor cores
            const uint32_t id_a = bf16_idesc(128, 0, 0), id_o = bf16_idesc(E, 0, 1);
            // descriptors count in 16 bytes: 16 values of a K-major tile, 16 ticks (rows) of an MN-major one
            constexpr auto along = [](int k) { return (uint64_t)((k >> 2) * (kBox >> 4) + (k & 3) * 2); };
            const uint64_t state_rows = swizzled(sm + L::state, kStateBox);
#pragma unroll 1
            for (int i = 0; i < chunks && ok; ++i) {
                const uint32_t stage = sm + (i & 1) * L::stage;
                const uint64_t a_ticks = swizzled(stage + L::a, 0), b_ticks = swizzled(stage + L::b, 0), c_rows = swizzled(stage + L::c, kBox);
                // W of the chunk before is read; and b' of it made, so that those who make it have seen its A
                ok = wait_full(i) && (i == 0 || (wait_stage(kPv0, i - 1) && (!L::own_terms || wait(kBReady, i - 1))));
                if (!ok) break;
                fg::tc_fence_after();
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) mma_bf16(tmem + tA, a_ticks + along(k), b_ticks + along(k), id_a, k > 0);
                fg::mma_commit(bar(kQk));
                ok = wait(kSReady, i) && (i == 0 || wait(kOutRead, i - 1));
                if (!ok) break;
                fg::tc_fence_after();
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) mma_bf16(tmem + tO1, a_ticks + along(k), state_rows + 128 * k, id_o, k > 0);
                fg::mma_commit(bar(kQs));
                ok = wait(kWReady, i) && (ticks_of(i) == kTcTicks || wait(kBReady, i));   // (c's end is cleared there)
                if (!ok) break;
                fg::tc_fence_after();
#pragma unroll
                for (int k = 0; k < kTcTicks / 16; ++k) mma_bf16_tmem(tmem + tO2, tmem + tA + k * 16, c_rows + 128 * k, id_o, k > 0);
                fg::mma_commit(bar(kPv0 + (i & 1)));
            }
        } else if (warp == 19 && lane == 0 && !PARTS) {
            // out of whole chunks, round by round
            constexpr int values = F32 ? 32 : 64;
            int round = 0;
#pragma unroll 1
            for (int i = 0; i < chunks && ok; ++i) {
                if (ticks_of(i) < kTcTicks) break;
#pragma unroll 1
                for (int e0 = 0; e0 < E && ok; e0 += kRound) {
                    ok = wait(kOutReady, round++);
                    if (!ok) break;
#pragma unroll 1
                    for (int e = e0; e < min(E, e0 + kRound); e += values)
                        tma_store(&maps.out, sm + out_at(i) + (e - e0) / values * kBox, e, h, first_of(i), batch);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    stores_read();
                    fg::mbar_arrive(bar(kOutStored));
                }
                if (!L::own_out && ok) fg::mbar_arrive(bar(kOutLeft0 + (i & 1)));
            }
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        } else if (warp == 18 && lane == 0) {
            // dS
            const uint32_t id_s = bf16_idesc(E, 1, 1);
            constexpr uint32_t next_b = DP == 128 ? kBox : 0;     // (an M = 128 operand of 64 values: twice the same)
            const uint64_t third = swizzled(sm + L::third, next_b);
#pragma unroll 1
            for (int i = 0; i < chunks && ok; ++i) {
                const uint32_t stage = sm + (i & 1) * L::stage;
                const uint64_t first = swizzled(stage + L::b, next_b), c_rows = swizzled(stage + L::c, kBox),
                               second = swizzled(L::own_terms ? sm + L::second : stage + L::a, next_b);
                ok = wait_full(i) && wait(kBReady, i) && wait(kSReady, i);   // dS of the chunk before has been read
                if (!ok) break;
                fg::tc_fence_after();
#pragma unroll
                for (int k = 0; k < 8; ++k) mma_bf16(tmem + tS, first + 128 * k, c_rows + 128 * k, id_s, k > 0);
#pragma unroll
                for (int k = 0; k < 8; ++k) mma_bf16(tmem + tS, second + 128 * k, c_rows + 128 * k, id_s, true);
#pragma unroll
                for (int k = 0; k < 8; ++k) mma_bf16(tmem + tS, third + 128 * k, c_rows + 128 * k, id_s, true);
                fg::mma_commit(bar(kKv0 + (i & 1)));
            }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // ---- ticks ---------------------------------------------------------------------------------------------
        const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        // gamma^{t-s} of a block of 16 columns s0 .. is gamma^{t-s0-15} gamma^{15-j} (from the back gamma^{s0-t} gamma^j). Off the
        // diagonal both are at most 1; on it the first may be over 1, and where it could overflow the weights are looked up.
        uint64_t near[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) near[k] = BACK ? two(pw[2 * k], pw[2 * k + 1]) : two(pw[15 - 2 * k], pw[14 - 2 * k]);
        const float scale = s.scale_in * s.scale_out;
        const bool in_range = ld > -2.f;                     // (e^(2 * 31) is finite by far)
        int round = 0;
#pragma unroll 1
        for (int i = 0; !PARTS && i < chunks && ok; ++i) {
            const int n = ticks_of(i);
            ok = together(wait(kQk, i));
            if (!ok) break;
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
                const int blk = (j & 2) + half, s0 = blk * 32 + (j & 1) * 16;   // blocks of 32 on one side of the diagonal are 0
                uint32_t v[16], x[8];
                if (BACK ? blk < quarter : blk > quarter) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = 0;
                    tmem_st8(lanes + tA + s0, x);
                    continue;
                }
                tmem_ld16(lanes + tA + s0, v);
                const int away = BACK ? s0 - row : row - s0 - 15;   // exponent of the first factor
                const float e = (in_range ? expf(ld * (float)away) : power(ld, (float)away)) * scale;
                tmem_ready(v);
                if (blk != quarter || in_range) {
                    const uint64_t e2 = two(e, e);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        x[k] = pack2(mul2(two(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), mul2(e2, near[k])));
                } else {                                      // (rare: one pair at a time, to keep it short)
#pragma unroll 1
                    for (int k = 0; k < 16; k += 2) {
                        const float* g = pw + (BACK ? s0 + k - row : row - s0 - k);   // gamma^{t-s}; 0 past the diagonal
                        const uint32_t y = pack_bf16(__uint_as_float(v[0]) * g[0] * scale, __uint_as_float(v[1]) * g[BACK ? 1 : -1] * scale);
#pragma unroll
                        for (int m = 0; m < 14; ++m) v[m] = v[m + 2];
#pragma unroll
                        for (int m = 0; m < 7; ++m) x[m] = x[m + 1];
                        x[7] = y;
                    }
                }
                if (blk == quarter || (BACK && n < kTcTicks)) {
                    // only columns up to the diagonal (from it on), and only the chunk's own
                    const int lo = BACK ? row - s0 : 0, up = BACK ? n - s0 : row - s0 + 1;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t keep = (2 * k >= lo && 2 * k < up ? 0xffffu : 0u) | (2 * k + 1 >= lo && 2 * k + 1 < up ? 0xffff0000u : 0u);
                        x[k] &= keep;
                    }
                }
                tmem_st8(lanes + tA + s0, x);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fg::tc_fence_before();
            arrive(kWReady);
            ok = together(wait(kQs, i) && wait_stage(kPv0, i));
            if (!ok) break;
            // out of whole chunks is put together in shared memory and stored as tiles (a thread's own stores, 32 lines at a
            // time, held up the MMAs' operands); a recording's last ticks go by themselves: what follows them is another's
            const float f = pw[max(BACK ? n - 1 - row : row, 0) + (i ? 1 : lead0)] * s.scale_out;
            const uint64_t f2 = two(f, f);
            constexpr int units = F32 ? 4 : 2;                // 16-byte units of 16 columns
            auto out16 = [&](int e0, uint32_t (&x)[16]) {
                uint32_t y[16];
                tmem_ld16(lanes + tO1 + e0, x);
                tmem_ld16(lanes + tO2 + e0, y);
                tmem_ready(x);
                tmem_ready(y);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint64_t o = fma2(two(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), f2,
                                            two(__uint_as_float(y[2 * k]), __uint_as_float(y[2 * k + 1])));
                    if (F32) asm("mov.b64 {%0, %1}, %2;" : "=r"(x[2 * k]), "=r"(x[2 * k + 1]) : "l"(o));
                    else x[k] = pack2(o);
                }
            };
            auto put = [&](int e0, const uint32_t* x) {       // e0: column of the round
                const int u0 = e0 * units / 16;
                unsigned char* to = smem + out_at(i) + (u0 >> 3) * kBox + row * 128;
#pragma unroll
                for (int k = 0; k < units; ++k)
                    *reinterpret_cast<uint4*>(to + ((((u0 & 7) + k) ^ (row & 7)) << 4)) =
                        make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
            };
            auto done = [&]() {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(kOutReady);
            };
            if (n < kTcTicks) {
                const long long at = batch * s.out.batch + (long long)(first_of(i) + row) * s.out.tick + h * s.out.head;
#pragma unroll 1
                for (int e0 = half * 16; e0 < E; e0 += 32) {
                    uint32_t x[16];
                    out16(e0, x);
                    uint4* to = reinterpret_cast<uint4*>(s.out.p + (at + e0) * (F32 ? 4 : 2));
                    if (row < n) {
#pragma unroll
                        for (int k = 0; k < units; ++k) to[k] = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                    }
                    __syncwarp();
                }
                fg::tc_fence_before();
                arrive(kOutRead);
            } else if (L::own_out || F32) {
#pragma unroll 1
                for (int e0 = 0; e0 < E && ok; e0 += kRound, ++round) {
                    // the place is free: over c, once dS is done with it; the round before is stored
                    ok = together((L::own_out || e0 || wait_stage(kKv0, i)) && (!round || wait(kOutStored, round - 1)));
                    if (!ok) break;
#pragma unroll 1
                    for (int e = half * 16; e < min(E - e0, kRound); e += 32) {
                        uint32_t x[16];
                        out16(e0 + e, x);
                        put(e, x);
                    }
                    if (e0 + kRound >= E) {
                        fg::tc_fence_before();
                        arrive(kOutRead);
                    }
                    done();
                }
            } else {                                          // (read at once, so that the next chunk's O1 can come)
                uint32_t held[EP / 32][8];
#pragma unroll
                for (int j = 0; j < EP / 32; ++j) {
                    if ((2 * j + half) * 16 >= E) continue;
                    uint32_t x[16];
                    out16((2 * j + half) * 16, x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) held[j][k] = x[k];
                }
                fg::tc_fence_before();
                arrive(kOutRead);
                ok = together(wait_stage(kKv0, i) && (!i || wait(kOutStored, i - 1)));   // (a round a chunk)
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < EP / 32; ++j)
                    if ((2 * j + half) * 16 < E) put((2 * j + half) * 16, held[j]);
                done();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        // ---- state ---------------------------------------------------------------------------------------------
        const int quarter = warp & 3, half = (warp >> 2) & 1, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const bool mine = row < D;
        float S[EP / 32][16];
#pragma unroll
        for (int j = 0; j < EP / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) S[j][i] = 0.f;
        const long long state0 = ((long long)b * s.heads + h) * D * E;
        // S += f * the state at p, which may lie [E][D]
        auto add = [&](const float* p, float f, bool across) {
#pragma unroll
            for (int j = 0; j < EP / 32; ++j) {
                const int e0 = (2 * j + half) * 16;
                if (!mine || e0 >= E) continue;
                if (across) {
                    const float* q = p + (long long)e0 * D + row;
#pragma unroll
                    for (int i = 0; i < 16; ++i, q += D) S[j][i] = fmaf(f, *q, S[j][i]);
                } else {
                    const float4* q = reinterpret_cast<const float4*>(p + row * E + e0);
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
        };
        if (!PARTS) {
            const float* parts = s.partial + ((long long)b * s.heads + h) * s.parts * D * E;
#pragma unroll 1
            for (int p = s.first ? -1 : 0; p < part; ++p)
                add(p < 0 ? s.first + state0 : parts + (long long)p * D * E,
                    power(ld, (float)(p < 0 ? (BACK ? max(t0 - 1, 0ll) : t0) : t0 - min(sp.n, (p + 1) * per))), p < 0 && s.first_t);
        }
#pragma unroll 1
        for (int i = 0; i < chunks && ok; ++i) {
            // S as the operand of O1: rows d, columns e, swizzled (rows past D: zeros, for the k-steps of 16 up to DP), once
            // O1 of the chunk before is done with it (at 128, kQs is waited for below)
            if (!PARTS && L::own_terms && i) ok = together(wait(kQs, i - 1));
            if (!ok) break;
            if (!PARTS && row < DP) {
                unsigned char* at = smem + L::state + row * 128;
#pragma unroll
                for (int j = 0; j < EP / 32; ++j) {
                    const int e0 = (2 * j + half) * 16;
                    if (e0 >= E) continue;
                    const float* x = S[j];
#pragma unroll
                    for (int k = 0; k < 2; ++k, x += 8)
                        *reinterpret_cast<uint4*>(at + (e0 >> 6) * kStateBox + (((((e0 & 63) >> 3) + k) ^ (row & 7)) << 4)) =
                            make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            fg::tc_fence_before();
            arrive(kSReady);
            const int n = ticks_of(i);
            ok = together(b_free(i));
            if (!ok) break;
            fade_b(i, n, tid - 256);
            ok = together(wait_stage(kKv0, i));
            if (!ok) break;
            const float fade = pw[n - 1 + (i ? 1 : lead0)];
#pragma unroll
            for (int j = 0; j < EP / 32; ++j) {
                if ((2 * j + half) * 16 >= E) continue;
                uint32_t v[16];
                tmem_ld16(lanes + tS + (2 * j + half) * 16, v);
                tmem_ready(v);
#pragma unroll
                for (int k = 0; k < 16; ++k) S[j][k] = fmaf(S[j][k], fade, __uint_as_float(v[k]));
            }
        }
        float* to = PARTS ? s.partial + (((long long)b * s.heads + h) * s.parts + part) * D * E : hand_on ? s.last + state0 : nullptr;
        if (to && mine) {
            const bool across = !PARTS && s.last_t;
            // (a wait that ran out shows in what is handed on and, below, in all of out)
            const float f = *gave_up ? __int_as_float(0x7fc00000) : !PARTS && BACK && sp.n ? pw[1] : 1.f;
#pragma unroll
            for (int j = 0; j < EP / 32; ++j) {
                const int e0 = (2 * j + half) * 16;
                if (e0 >= E) continue;
                if (across) {
                    float* p = to + (long long)e0 * D + row;
#pragma unroll
                    for (int k = 0; k < 16; ++k, p += D) *p = f * S[j][k];
                } else {
                    float4* p = reinterpret_cast<float4*>(to + row * E + e0);
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
    if (!PARTS && warp >= 8 && warp < 16 && *gave_up) {       // (all stores are over: warp 19 has waited for its own)
        // the block's place anew: kept, it would cost every role registers
        int x, y;
        asm volatile("mov.u32 %0, %%ctaid.x;\n\tmov.u32 %1, %%ctaid.y;" : "=r"(x), "=r"(y));
        const Span all = span_of(s, x / s.heads);
        const long long size = part_ticks(all.n, s.parts), from = min(all.n, y * size), to = min(all.n, from + size);
        const long long at = (s.offsets ? 0 : x / s.heads) * s.out.batch + (x % s.heads) * s.out.head;
#pragma unroll 1
        for (long long t = from + warp - 8; t < to; t += 8)
#pragma unroll 1
            for (int e = lane; e < E; e += 32) {
                const long long i = at + (all.start + (BACK ? all.n - 1 - t : t)) * s.out.tick + e;
                if (F32) reinterpret_cast<uint32_t*>(s.out.p)[i] = 0x7fc00000u;
                else reinterpret_cast<uint16_t*>(s.out.p)[i] = 0x7fc0;
            }
    }
    if (last_block) wait_for_previous();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
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
           whole_units(s, s.out) && reinterpret_cast<uintptr_t>(s.last) % 16 == 0 &&
           (s.first_t || reinterpret_cast<uintptr_t>(s.first) % 16 == 0);   // (read value by value where it lies [E][D])
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
template <int DP, int EP, bool BACK, bool F32>
void tc_launch_as(const Scan& s, cudaStream_t st) {
    constexpr int bytes = TcLayout<DP, EP>::bytes;
    static OnEachDevice here;
    here.first(current_device(), [] {
        allow_shared(k_decay_tc<DP, EP, BACK, F32, false>, bytes);
        allow_shared(k_decay_tc<DP, EP, BACK, false, true>, bytes);
    });
    const TcMaps maps{tile_map(s, s.a, s.D), tile_map(s, s.b, s.D), tile_map(s, s.c, s.E), tile_map(s, s.out, s.E, F32)};
    const unsigned rows = (unsigned)(s.batch * s.heads);
    if (s.parts > 1) k_decay_tc<DP, EP, BACK, false, true><<<dim3(rows, s.parts - 1), kTcThreads, bytes, st>>>(s, maps);
    launch_beside(k_decay_tc<DP, EP, BACK, F32, false>, dim3(rows, s.parts), kTcThreads, bytes, st, s, maps);
}
template <bool BACK, bool F32>
void tc_launch_dims(const Scan& s, cudaStream_t st) {
    if (s.D > 64) s.E > 64 ? tc_launch_as<128, 128, BACK, F32>(s, st) : tc_launch_as<128, 64, BACK, F32>(s, st);
    else s.E > 64 ? tc_launch_as<64, 128, BACK, F32>(s, st) : tc_launch_as<64, 64, BACK, F32>(s, st);
}
inline void tc_launch(const Scan& s, cudaStream_t st) {
    if (!s.backward) tc_launch_dims<false, false>(s, st);
    else s.out_f32 ? tc_launch_dims<true, true>(s, st) : tc_launch_dims<true, false>(s, st);
}

}  // namespace
