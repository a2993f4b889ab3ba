// The product kernel for FWD of 16-bit matrices on 16 bytes whose sums are short or whose tiles are few (opal_linear.h has the products
// and the operands' layouts): 128 x 256 tiles, four waves of 128 x 64, two blocks on a CU that know nothing of each other.
//
// With short sums the epilogue, which is bound by memory, is most of a tile; opal_linear_big.h's one block a CU does nothing else
// meanwhile.  Here what one block waits for (the first chunks of its tile, a barrier, the residual, its stores) the other fills with
// sums: 250 000 x 355 x 128 in 66 us, 2.6 TB/s and 346 TFLOP/s, against 82.  Long sums are bound by the chunks' way, and narrower tiles ask for
// more of them: 48 KB for 1024 cycles of the matrix pipes, where a CU takes 58 bytes a cycle; 250 000 x 512 x 1564 takes 500 us against 399.
//   - A wave reads the next 16 k while it multiplies the present ones; one barrier for each 32 k.
//   - Chunks come straight into LDS, two steps ahead.  A (from memory): 2 x 64 k, whole 128-byte lines, of which a CU has only so many on
//     their way; B (W stays in L2): 3 x 32 k.  32 + 48 KB, half of a CU's LDS.
//   - A block ends with its tile: the next one starts where a CU has room, and nothing waits for the stores.
#pragma once
#include "opal_linear_big.h"

namespace opal_head {

constexpr int PAIR_M = 128, PAIR_N = 256, PAIR_THREADS = 256;

// ROWS lines of K values of k a stage, N stages
template <int ROWS, int K_, int N_> struct PairSide {
    static constexpr int K = K_, N = N_, BYTES = ROWS * K * 2, LINE = K / 8, AT_ONCE = PAIR_THREADS / LINE, PARTS = ROWS / AT_ONCE;
    static_assert(PARTS == 4 && ROWS <= PAIR_THREADS && AT_ONCE % 16 == 0, "four requests a thread and stage; the rotation repeats after 16 lines");
    const char *p;                             // the first element of stage 0
    uint32_t ld, off, hop;                     // bytes
    int rows, lim;                             // lim: first k of this thread's chunk

    // lines of 128 (64) bytes, two (four) of which share the banks: the rotation gives a chunk of 16 lines 16 places
    __device__ __forceinline__ static int swz(int line) { return K == 64 ? swizzle_kc(line) : (line >> 2) & 3; }
    __device__ __forceinline__ void init(const char *base, uint64_t stride, uint64_t first, uint64_t end)
    {
        const int t = threadIdx.x, line = t / LINE, chunk = (t % LINE) ^ swz(line);
        ld = (uint32_t)stride * 2;
        p = base + first * ld;
        rows = (int)(end - first < (uint64_t)ROWS ? end - first : (uint64_t)ROWS);
        off = line * ld + chunk * 16;
        hop = AT_ONCE * ld;
        lim = chunk * 8;
    }
    // A quarter of stage q of a sum of k values.  The buffer ends with the 16 bytes that hold the stage's last element (nothing of a
    // stage behind the sum's end): lines and chunks behind read as zeros.
    __device__ __forceinline__ void request(char *lds, uint32_t q, uint32_t slot, uint32_t k, int part, int wave) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        const int left = (int)k - (int)(q * K), kval = left < K ? left : K;
        const uint32_t len = left > 0 ? ((uint32_t)(rows - 1) * ld + (uint32_t)kval * 2u + 15u) & ~15u : 0u;
        auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(p + (uint64_t)q * (K * 2)), (short)0, (int)len, 0x00020000);
        const uint32_t at = lim >= kval ? 0x80000000u : off + part * hop;       // behind every buffer (smaller than 2^31)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (OPAL_LDS void *)(lds + slot * BYTES + part * 4096 + wave * 1024), 16, (int)at, 0, 0, 0);
#endif
    }
    // The k behind the sum's end in the chunk that holds it (k: of the stage; not a multiple of eight).
    __device__ __forceinline__ static void clear(char *lds, int k)
    {
        const int r = threadIdx.x;
        if (r >= ROWS) return;
        uint16_t *c = reinterpret_cast<uint16_t *>(lds + r * (K * 2) + (((k >> 3) ^ swz(r)) * 16));
        for (int e = k & 7; e < 8; e++) c[e] = 0;
    }
    // fragments of COUNT times 32 lines from r0 on and the 16 k from 16 kk on: k = 8 (lane / 32) + 0..7
    template <int COUNT> __device__ __forceinline__ static void frags(const char *lds, int r0, int kk, s16x8 (&f)[COUNT])
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            const int r = r0 + i * 32 + (lane & 31), c = kk * 2 + (lane >> 5);
            f[i] = *reinterpret_cast<const s16x8 *>(lds + r * (K * 2) + ((c ^ swz(r)) * 16));
        }
    }
};

template <class T, int ACT, bool Y32, int RES> __global__ __launch_bounds__(PAIR_THREADS, 2) void linear_pair_kernel(const Linear g)
{
    using SA = PairSide<PAIR_M, 64, 2>;
    using SB = PairSide<PAIR_N, 32, 3>;
    __shared__ __attribute__((aligned(128))) char lds[SA::N * SA::BYTES + SB::N * SB::BYTES];
    char *const lb = lds + SA::N * SA::BYTES;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave * 64;
    const uint32_t t = xcd_tile(blockIdx.x, gridDim.x), tm = t / g.tn, tn = t - tm * g.tn;
    const uint32_t K = (uint32_t)g.K;
    SA a;
    SB b;
    a.init(g.a, g.lda, (uint64_t)tm * PAIR_M, g.M);
    b.init(g.b, g.ldb, (uint64_t)tn * PAIR_N, g.N);
    const uint32_t steps = (K + 31) / 32;
    const int tail = (int)(K - (steps - 1) * 32);
    const uint32_t cut = tail & 7 ? steps - 1 : ~0u;            // the step whose k end inside a chunk
#pragma unroll
    for (int i = 0; i < 4; i++) b.request(lb, 0, 0, K, i, wave);
#pragma unroll
    for (int i = 0; i < 4; i++) a.request(lds, 0, 0, K, i, wave);
#pragma unroll
    for (int i = 0; i < 4; i++) b.request(lb, 1, 1, K, i, wave);
#pragma unroll
    for (int i = 0; i < 4; i++) b.request(lb, 2, 2, K, i, wave);
#pragma unroll
    for (int i = 0; i < 4; i++) a.request(lds, 1, 1, K, i, wave);
    if ((uint64_t)tn * PAIR_N + wn >= g.N) {   // a wave without columns has its share of the requests to make, and nothing else
        asm volatile("s_waitcnt vmcnt(12)\n\ts_barrier" ::: "memory");
        uint32_t slot_a = 0, slot_b = 0;
        if (cut == 0) {
            SA::clear(lds, tail);
            SB::clear(lb, tail);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll 1
        for (uint32_t s = 0; s < (steps + 1) / 2 * 2; s++) {
            const uint32_t o = s & 1, next_b = slot_b + 1 == SB::N ? 0 : slot_b + 1, next_a = slot_a ^ o;
            if (o) asm volatile("s_waitcnt vmcnt(4)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
            if (s + 1 == cut) {
                SA::clear(lds + next_a * SA::BYTES, tail + (o ? 0 : 32));
                SB::clear(lb + next_b * SB::BYTES, tail);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            for (int i = 0; i < 4; i++) b.request(lb, s + 3, slot_b, K, i, wave);
            if (o)
                for (int i = 0; i < 4; i++) a.request(lds, s / 2 + 2, slot_a, K, i, wave);
            slot_a = next_a;
            slot_b = next_b;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        return;
    }
    f32x16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
    asm volatile("s_waitcnt vmcnt(12)\n\ts_barrier" ::: "memory");
    s16x8 fa[2][4], fb[2][2];
    if (cut == 0) {
        SA::clear(lds, tail);
        SB::clear(lb, tail);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    SA::template frags<4>(lds, 0, 0, fa[0]);
    SB::template frags<2>(lb, wn, 0, fb[0]);
    uint32_t slot_a = 0, slot_b = 0;           // of the present step
    // At a step's barrier its fragments are all read, and the next step's chunks have arrived: what was asked for behind them may be
    // on its way still, which is B of the step after next and, in A's even steps, A's next stage.  A sum of an odd number of steps
    // ends with one of zeros.
#pragma unroll 1
    for (uint32_t s0 = 0; s0 < steps; s0 += 2, slot_a ^= 1) {
#pragma unroll
        for (uint32_t o = 0; o < 2; o++) {
            const uint32_t s = s0 + o, next_b = slot_b + 1 == SB::N ? 0 : slot_b + 1, next_a = slot_a ^ o;
            SA::template frags<4>(lds + slot_a * SA::BYTES, 0, o * 2 + 1, fa[1]);
            SB::template frags<2>(lb + slot_b * SB::BYTES, wn, 1, fb[1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = mfma16<T>(fb[0][j], fa[0][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
            if (o) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 == cut) {
                SA::clear(lds + next_a * SA::BYTES, tail + (o ? 0 : 32));
                SB::clear(lb + next_b * SB::BYTES, tail);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            SA::template frags<4>(lds + next_a * SA::BYTES, 0, o ? 0 : 2, fa[0]);
            SB::template frags<2>(lb + next_b * SB::BYTES, wn, 0, fb[0]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = mfma16<T>(fb[1][j], fa[1][i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
                b.request(lb, s + 3, slot_b, K, i, wave);
                if (o) a.request(lds, s / 2 + 2, slot_a, K, i, wave);
                __builtin_amdgcn_sched_barrier(0);
            }
            slot_b = next_b;
        }
    }
    // what was asked for behind the end must not arrive in another block's LDS
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    BigItem c;
    c.m0 = tm * PAIR_M;
    c.n0 = tn * PAIR_N;
    c.split = 0;
    epilogue<T, FWD, ACT, Y32, RES>(g, c, acc, 0, wn, 0);
}

template <class T> hipError_t launch_pair(const Linear &g, hipStream_t stream)
{
    const int res = !g.res ? 0 : g.res_type == OPAL_F32 ? RES32 : RES16;
#define OPAL_PAIR(ACT, Y32, RES)                                                                                                     \
    if (g.act == ACT && (g.y_type == OPAL_F32) == Y32 && res == RES) {                                                                \
        hipLaunchKernelGGL((linear_pair_kernel<T, ACT, Y32, RES>), dim3(g.tm * g.tn), dim3(PAIR_THREADS), 0, stream, g);               \
        return hipGetLastError();                                                                                                    \
    }
#define OPAL_PAIRS(Y32, RES) OPAL_PAIR(ACT_NONE, Y32, RES) OPAL_PAIR(ACT_RELU, Y32, RES) OPAL_PAIR(ACT_SILU, Y32, RES) OPAL_PAIR(ACT_GELU, Y32, RES)
    OPAL_PAIRS(false, 0)
    OPAL_PAIRS(false, RES16)
    OPAL_PAIRS(false, RES32)
    OPAL_PAIRS(true, 0)
    OPAL_PAIRS(true, RES16)
    OPAL_PAIRS(true, RES32)
#undef OPAL_PAIRS
#undef OPAL_PAIR
    return hipErrorInvalidValue;
}

}  // namespace opal_head
