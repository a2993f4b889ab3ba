// The product kernel for large 16-bit matrices on 16 bytes (opal_linear.h has the products, the operands' layouts and the kernel
// for everything else): 256 x 256 tiles, eight waves of 128 x 64, one block per CU that stays for all its tiles, steps of 32 k.
//
// What bounds it: a half's turn at the matrix pipe (16 MFMAs, 512 cycles) against the other's reads meanwhile (48 KB of LDS at 125 bytes a
// cycle and their way), the way of the chunks (32 KB a step; a CU takes 58 bytes a cycle, without loss to its LDS reads), and the
// clock, which falls under the load.  Sums of the hidden layer's product (250 000 x 512 x 1564) 350 us, 1146 TFLOP/s; with all operands zero 306; with
// the epilogue 399, with bias, GELU and the value before it 470.  Input gradient 100 000 x 512 x 1564 in float16 with GELU 207 us, weight
// gradient 1564 x 512 of 100 000 rows 185 us and 12 for the splits' sum.
//   - Waves 0 .. 3 and 4 .. 7 share the four SIMDs and take turns: while one half multiplies (16 MFMAs, its requests for chunks in
//     between), the other reads its next fragments, with a barrier at each change; half 1 runs one change behind half 0.
//   - Chunks come straight into LDS, well ahead and over the ends of tiles.  Half 0 asks for A's, half 1 for B's: vmcnt counts a
//     wave's requests in their order, so A's long way (memory) and B's short one (W stays in L2) must not share a count.
//   - A of FWD and GIN is fetched 64 k at a time: whole 128-byte lines, of which a CU has only so many on their way.
//   - The epilogue works in the accumulators' own places; its stores drain under the next tile's steps.
#pragma once
#include "opal_linear.h"

namespace opal_head {

constexpr int BIG = 256, BIG_THREADS = 512, BIG_STEP = 32;

// k per stage and stages of an operand's ring.  FWD, GIN: A 3 x 64 k (96 KB), B 3 x 32 k (48 KB); GWT, whose operands both come
// from memory in whole lines (MC): 4 x 32 k each (128 KB).  Each of a half's four waves asks for four chunks a lane and step.
//
// When a stage's place is free: both halves have read stage s once half 1 multiplies it (it reads after half 0), which is when half 1
// asks for B's stage s + N; half 0, which asks for A, multiplies one change earlier and may only refill the place of the stage before:
// A's stage s + N - 1.
template <int P, bool IS_A> struct Ring {
    static constexpr bool KC = IS_A ? P != GWT : P == FWD;
    static constexpr int K = P != GWT && IS_A ? 64 : 32, N = P == GWT ? 4 : 3;
    static constexpr int BYTES = BIG * K * 2, PARTS = K / BIG_STEP, AHEAD = IS_A ? N - 1 : N;
    static constexpr int WAIT = (N - 2) * 4 * PARTS;                          // requests that may be on their way behind the next stage's
    static constexpr int LINE = KC ? K / 8 : 32;                              // chunks: KC has 256 lines, MC one for each k
    // KC: lines of 128 (64) bytes, two (four) of which share the banks: the rotation gives a chunk of 16 rows 16 places
    __device__ __forceinline__ static int swz(int line) { return !KC ? swizzle_mc<2, BIG>(line) : K == 64 ? swizzle_kc(line) : (line >> 2) & 3; }
    // bytes from a stage's first element on that are the matrix's, up to the end of the 16 that hold the last one; lines behind read as zeros
    __device__ __forceinline__ static uint32_t length(uint32_t ld, int rows, int kval)
    {
        return ((uint32_t)((KC ? rows : kval) - 1) * ld + (uint32_t)(KC ? kval : rows) * 2u + 15u) & ~15u;
    }
    // Fragments of COUNT times 32 rows from r0 on, the block `rot` first, and of the 32 k that begin at 16 kk: k = 8 (lane / 32) + 0..7 of 16.
    template <int COUNT> __device__ __forceinline__ static void frags(const char *lds, int r0, int rot, int kk, s16x8 (&f)[2][COUNT])
    {
        const int lane = threadIdx.x & 63;
        if constexpr (KC) {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < COUNT; i++) {
                    const int r = r0 + i * 32 + (lane & 31), c = (kk + s) * 2 + (lane >> 5);
                    f[s][i] = *reinterpret_cast<const s16x8 *>(lds + r * (K * 2) + ((c ^ swz(r)) * 16));
                }
        } else {
#pragma unroll
            for (int i = 0; i < COUNT; i += 2) {
                uint64_t x[8];
                read_tr8<4 * BIG * 2, 16 * BIG * 2>(lds_place(lds) + tr_place<BIG>(r0 + ((i + rot) & (COUNT - 1)) * 32),
                                                     lds_place(lds) + tr_place<BIG>(r0 + ((i + 1 + rot) & (COUNT - 1)) * 32), x);
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    f[s][i] = join_tr(x[2 * s], x[2 * s + 1]);
                    f[s][i + 1] = join_tr(x[4 + 2 * s], x[5 + 2 * s]);
                }
            }
        }
    }
};
constexpr int RES16 = 1, RES32 = 2;            // kinds of residual: the operands' type, 32 bits

// the k of a KC fragment behind the matrix's edge: `left` values of k from the fragment's first on are the matrix's
__device__ __forceinline__ s16x8 keep_k(s16x8 f, int left)
{
    u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = left >= 2 * i + 2 ? w[i] : left == 2 * i + 1 ? w[i] & 0xffffu : 0u;
    return __builtin_bit_cast(s16x8, w);
}

struct BigItem {                               // one tile (of one split)
    uint32_t m0, n0, split;
    int rows_a, rows_b;
    uint64_t k, count;                         // first k, number of k
};
template <int P> __device__ __forceinline__ BigItem big_item(const Linear &g, uint32_t i)
{
    uint32_t t = xcd_tile(i, g.items);
    const uint32_t tiles = g.tm * g.tn, split = P == GWT ? t / tiles : 0;
    t -= split * tiles;
    BigItem r;
    const uint32_t tm = t / g.tn, tn = t - tm * g.tn;
    r.m0 = tm * BIG;
    r.n0 = tn * BIG;
    r.split = split;
    r.rows_a = (int)(g.M - r.m0 < (uint64_t)BIG ? g.M - r.m0 : (uint64_t)BIG);
    r.rows_b = (int)(g.N - r.n0 < (uint64_t)BIG ? g.N - r.n0 : (uint64_t)BIG);
    r.k = split * g.ksplit;
    r.count = (P == GWT && r.k + g.ksplit < g.K ? r.k + g.ksplit : g.K) - r.k;
    return r;
}

// The launch's description, read again from the argument segment (a few hundred cycles, once a tile) rather than kept in scalar
// registers through the loop, where there are none to spare.
__device__ __forceinline__ const Linear &reload()
{
#ifdef __HIP_DEVICE_COMPILE__
    auto p = (const __attribute__((address_space(4))) Linear *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Linear *)p;
#else
    __builtin_unreachable();
#endif
}

// A wave's requests: half 0 feeds A, half 1 B.  The two differ in numbers only, so that a request is the same instruction for both.
template <int P> struct Feed {
    using RA = Ring<P, true>;
    using RB = Ring<P, false>;
    const char *p;                             // the next stage's first element
    uint64_t step;
    uint32_t off, hop, ring, item, slot, left, len, last;
    uint32_t at, now, to;                      // of the requests at hand
    int lim, tail, half;                       // lim: first k of this thread's chunks (KC), -1 where the end of k cuts lines (MC)

    __device__ __forceinline__ void init(int wave)
    {
        const Linear &g = reload();
        half = wave >> 2;
        const uint32_t t = threadIdx.x & 255;
        place<RA>(g.lda, half == 0, t);
        place<RB>(g.ldb, half == 1, t);
        ring = (half ? RA::N * RA::BYTES : 0) + (wave & 3) * 1024;
        item = blockIdx.x;
        slot = 0;
        open();
    }
    template <class R> __device__ __forceinline__ void place(uint64_t elements, bool mine, uint32_t t)
    {
        static_assert((256 / R::LINE) % 16 == 0 || !R::KC, "the rotation repeats after 16 lines");
        if (!mine) return;
        const uint32_t ld = (uint32_t)elements * 2, line = t / R::LINE, chunk = (t % R::LINE) ^ R::swz(line);
        off = line * ld + chunk * 16;
        hop = 256 / R::LINE * ld;              // whole rotations further: the same place in the line
        lim = R::KC ? (int)chunk * 8 : -1;
        step = R::KC ? R::K * 2 : (uint64_t)R::K * ld;
    }
    // Turns to the tile `item`; behind the last one to an empty buffer (zeros that nobody reads): every stage has the same requests.
    __device__ __forceinline__ void open()
    {
        const Linear &g = reload();
        const bool any = item < g.items;
        const BigItem f = big_item<P>(g, any ? item : 0);
        if (half == 0) aim<RA>(g.a, g.lda * 2, f.m0, f.rows_a, f, any);
        else aim<RB>(g.b, g.ldb * 2, f.n0, f.rows_b, f, any);
    }
    template <class R> __device__ __forceinline__ void aim(const char *matrix, uint64_t ld, uint64_t first, int rows, const BigItem &f, bool any)
    {
        const uint32_t stages = (uint32_t)((f.count + R::K - 1) / R::K);
        p = matrix + (R::KC ? first * ld + f.k * 2 : f.k * ld + first * 2);
        tail = any ? (int)(f.count - (uint64_t)(stages - 1) * R::K) : R::K;
        left = any ? stages : 0x7fffffffu;
        len = any ? R::length((uint32_t)ld, rows, R::K) : 0;
        last = any ? R::length((uint32_t)ld, rows, tail) : 0;
    }
    // the requests of a step: `part` of the stage, 0 .. PARTS - 1
    __device__ __forceinline__ void start(int part)
    {
        at = left == 1 && lim >= tail ? 0x80000000u : off;       // behind every buffer (smaller than 2^31)
        at += part * 4 * hop;
        now = left == 1 ? last : len;
        to = ring + slot * (half ? RB::BYTES : RA::BYTES) + part * 4 * 4096;
    }
    __device__ __forceinline__ void request(char *lds, int i) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, (int)now, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (OPAL_LDS void *)(lds + to + i * 4096), 16, (int)(at + i * hop), 0, 0, 0);
#endif
    }
    __device__ __forceinline__ void done()     // the stage is asked for
    {
        slot = slot + 1 == (uint32_t)RA::N ? 0 : slot + 1;
        p += step;
        if (--left == 0) {
            item += reload().blocks;
            open();
        }
    }
    __device__ __forceinline__ void stage(char *lds)
    {
        for (int part = 0; part < (half ? RB::PARTS : RA::PARTS); part++) {
            start(part);
            for (int i = 0; i < 4; i++) request(lds, i);
        }
        done();
    }
};

// ------------------------------------------------------------------------------------------------ epilogue

// An accumulator's 32 x 32 results: a lane holds row l % 32 and of each group of eight columns four, 16 bytes (8 in 16 bits) here and
// there.  What a wave writes at once should be long pieces of rows, so two exchanges of lanes put columns where rows were:
//   by 16 lanes: a lane holds rows l % 16 and l % 16 + 16, and four columns of each 16: 4 lanes make 64 bytes of a row in 32 bits
//   by 32 lanes (16-bit results only): eight columns of 32: 4 lanes make 64 bytes of a row
template <int LANES> __device__ __forceinline__ void exchange(uint32_t &x, uint32_t &y)
{
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (LANES == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        x = r[0];
        y = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        x = r[0];
        y = r[1];
    }
#endif
}
// v[8 u + 4 R + e] afterwards: row 16 R + l % 16, column 16 u + 8 (l / 16 % 2) + 4 (l / 32) + e
__device__ __forceinline__ void turn16(f32x16 &v)
{
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = v[u * 8 + e], b = v[u * 8 + 4 + e];
            uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
            exchange<16>(x, y);
            v[u * 8 + e] = __builtin_bit_cast(float, x);
            v[u * 8 + 4 + e] = __builtin_bit_cast(float, y);
        }
}
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    struct H { T v[2]; } h = {{(T)a, (T)b}};
    return __builtin_bit_cast(uint32_t, h);
}
struct __attribute__((packed, aligned(2))) Any16 { uint32_t w[4]; };

// row R's eight columns from 16 (l / 32) + 8 (l / 16 % 2) on, of a turned block; `left` of them the matrix's
template <class T> __device__ __forceinline__ void store_joined(void *to, uint64_t at, int left, const f32x16 &v, int R)
{
    uint32_t x0 = pack2<T>(v[R * 4], v[R * 4 + 1]), x1 = pack2<T>(v[R * 4 + 2], v[R * 4 + 3]);
    uint32_t y0 = pack2<T>(v[8 + R * 4], v[8 + R * 4 + 1]), y1 = pack2<T>(v[8 + R * 4 + 2], v[8 + R * 4 + 3]);
    exchange<32>(x0, y0);
    exchange<32>(x1, y1);
    const Any16 o = {{x0, x1, y0, y1}};
    if (left >= 8) *reinterpret_cast<Any16 *>((T *)to + at) = o;
    else
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < left) ((uint16_t *)to)[at + e] = (uint16_t)(o.w[e / 2] >> (16 * (e & 1)));
}
// the same places of a matrix that is read: eight columns of row R as they lie in memory, and (exchanged back) as the turned block has them
__device__ __forceinline__ Any16 load_joined(const void *from, uint64_t at, int left)
{
    Any16 r = {{0, 0, 0, 0}};
    if (left >= 8) r = *reinterpret_cast<const Any16 *>((const uint16_t *)from + at);
    else
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < left) r.w[e / 2] |= (uint32_t)((const uint16_t *)from)[at + e] << (16 * (e & 1));
    return r;
}
template <class T> __device__ __forceinline__ void part_joined(const Any16 &r, f32x4 (&c)[2])      // c[u]: columns of the u-th 16
{
    uint32_t x0 = r.w[0], x1 = r.w[1], y0 = r.w[2], y1 = r.w[3];
    exchange<32>(x0, y0);
    exchange<32>(x1, y1);
    struct Q { T v[4]; };
    struct W { uint32_t a, b; };
    const Q p = __builtin_bit_cast(Q, (W{x0, x1})), q = __builtin_bit_cast(Q, (W{y0, y1}));
#pragma unroll
    for (int e = 0; e < 4; e++) {
        c[0][e] = (float)p.v[e];
        c[1][e] = (float)q.v[e];
    }
}

// 32 x 32 results at a time, straight from the accumulators.  What is read is asked for ahead, all of a 16-bit residual first (60 001 x 1563 x
// 512 254 -> 240 us).  Results in 32 bits (Y32) or the operands' type; a residual in 32 bits (RES32) or the operands' type (RES16).
template <class T, int P, int ACT, bool Y32, int RES>
__device__ __forceinline__ void epilogue(const Linear &g, const BigItem &c, const f32x16 (&acc)[4][2], int wm, int wn, int rot)
{
    const int lane = threadIdx.x & 63, h = lane >> 5, b4 = (lane >> 4) & 1;
    const uint32_t m0 = c.m0 + wm + (lane & 15), n0 = c.n0 + wn, N = (uint32_t)g.N, M = (uint32_t)g.M;
    const uint32_t nq = n0 + b4 * 8 + h * 4, nj = n0 + h * 16 + b4 * 8;       // this lane's columns: four of each 16, and eight of 32
    constexpr bool with_pre = P == GIN && ACT;                 // known here: a load that might not be used would be waited for in the loop
    constexpr int AHEAD = RES == RES16 && !with_pre ? 7 : 1, RING = AHEAD + 1;       // blocks asked for ahead: all where registers allow
    f32x4 res32[RES == RES32 ? RING : 1][2][2];
    Any16 res16[RES == RES16 ? RING : 1][2], pre[with_pre ? RING : 1][2];
    auto ask = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int R = 0; R < 2; R++) {
            const uint32_t m = m0 + (((t >> 1) + rot) & 3) * 32 + R * 16, n = nj + (t & 1) * 32;
            if constexpr (RES == RES32)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t at = nq + (t & 1) * 32 + u * 16;
                    res32[t % RING][R][u] = load4_typed(g.res, OPAL_F32, m * g.ldr + at, m < M ? (int)(N - at) : 0);
                }
            if constexpr (RES == RES16) res16[t % RING][R] = load_joined(g.res, m * g.ldr + n, m < M ? (int)(N - n) : 0);
            if constexpr (with_pre) pre[t % RING][R] = load_joined(g.pre_in, m * g.ldp + n, m < M ? (int)(N - n) : 0);
        }
    };
    if (RES || with_pre)
#pragma unroll
        for (int t = 0; t < AHEAD; t++) ask(t);
    f32x4 bias[2][2] = {};
    if (P == FWD && g.bias)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                bias[j][u] = load4_typed(g.bias, OPAL_F32, nq + j * 32 + u * 16, (int)(N - (nq + j * 32 + u * 16)));
#pragma unroll
    for (int t = 0; t < 8; t++) {
        f32x16 v = acc[t >> 1][t & 1];
        if ((RES || with_pre) && t + AHEAD < 8) ask(t + AHEAD);
        turn16(v);
        if (P == FWD) {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] += bias[t & 1][e >> 3][e & 3];
        }
        const uint32_t m = m0 + (((t >> 1) + rot) & 3) * 32, n = nj + (t & 1) * 32;
        if (P == FWD && g.pre_out) {
#pragma unroll
            for (int R = 0; R < 2; R++) store_joined<T>(g.pre_out, (m + R * 16) * g.ldp + n, m + R * 16 < M ? (int)(N - n) : 0, v, R);
        }
        if (P == FWD && ACT) {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = act_value(v[e], ACT);
        }
#pragma unroll
        for (int R = 0; R < 2; R++) {
            if constexpr (with_pre) {
                f32x4 z[2];
                part_joined<T>(pre[t % RING][R], z);
#pragma unroll
                for (int e = 0; e < 8; e++) v[(e >> 2) * 8 + R * 4 + (e & 3)] *= act_slope(z[e >> 2][e & 3], ACT);
            }
            if constexpr (RES != 0) {
                f32x4 r[2];
                if constexpr (RES == RES32) {
                    r[0] = res32[t % RING][R][0];
                    r[1] = res32[t % RING][R][1];
                } else part_joined<T>(res16[t % RING][R], r);
#pragma unroll
                for (int e = 0; e < 8; e++) v[(e >> 2) * 8 + R * 4 + (e & 3)] += r[e >> 2][e & 3];
            }
            if constexpr (Y32) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t at = nq + (t & 1) * 32 + u * 16;
                    store4_typed(g.y, OPAL_F32, c.split * g.y_split + (m + R * 16) * g.ldy + at, m + R * 16 < M ? (int)(N - at) : 0,
                                 f32x4{v[u * 8 + R * 4], v[u * 8 + R * 4 + 1], v[u * 8 + R * 4 + 2], v[u * 8 + R * 4 + 3]});
                }
            } else store_joined<T>(g.y, (m + R * 16) * g.ldy + n, m + R * 16 < M ? (int)(N - n) : 0, v, R);
        }
    }
}

// ------------------------------------------------------------------------------------------------ main loop
// One step of a wave: fragments, the change of turns, 16 MFMAs and its requests.  CUT: the last step of a sum whose k end inside a
// chunk.  sub: the step's 32 k within A's stage.  fresh: the next step begins a new stage of A; last: of the tile.
template <class T, int P, bool CUT>
__device__ __forceinline__ void big_step(Feed<P> &feed, f32x16 (&acc)[4][2], char *lds, uint32_t slot_a, uint32_t slot_b, int sub, bool fresh, bool last, int wave,
                                         int half, int &landed, int ctail, bool sum_rows, float &colsum)
{
    using RA = Ring<P, true>;
    using RB = Ring<P, false>;
    const char *sa = lds + slot_a * RA::BYTES, *sb = lds + RA::N * RA::BYTES + slot_b * RB::BYTES;
    const int wm = half * 128, wn = (wave & 3) * 64;
    s16x8 fa[2][4], fb[2][2];
    RA::template frags<4>(sa, wm, P == GWT ? wave & 3 : 0, sub * 2, fa);
    RB::template frags<2>(sb, wn, 0, 0, fb);
    if (P == GWT && sum_rows) {                // of dy: this wave's first block, which its rotation makes another than its neighbours'
#pragma unroll
        for (int kk = 0; kk < 2; kk++) colsum += sum8<T>(fa[kk][0]);
    }
    if constexpr (CUT) {
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            const int left = ctail - kk * 16 - ((threadIdx.x >> 5) & 1) * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) fa[kk][i] = keep_k(fa[kk][i], left);
            if (P == FWD)
#pragma unroll
                for (int j = 0; j < 2; j++) fb[kk][j] = keep_k(fb[kk][j], left);
        }
    }
    const int part = half ? 0 : sub;
    feed.start(part);
    // The next stage has to be there before the barrier that opens it for half 0: half 1's requests here, half 0's behind its MFMAs.
    // vmcnt counts stores too, which an epilogue leaves behind; it waits for what was asked for before it, so that the next stages
    // need not wait for its stores (landed).
    if (half) {
        if (landed > 0) landed--;
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(RB::WAIT) : "memory");
    }
    // Between the two barriers of a turn stands nothing but MFMAs and, in their shadow, the requests (one for four of them).
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < 2; kk++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = mfma16<T>(fb[kk][j], fa[kk][i], acc[i][j]);
            if ((i & 1) == 0) {
                __builtin_amdgcn_sched_barrier(0);
                feed.request(lds, kk * 2 + i / 2);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    if (!half) {
        if (fresh) {
            if (sub < RA::PARTS - 1) {         // a tile that ends inside a stage: the rest of the requests
                feed.start(sub + 1);
                for (int i = 0; i < 4; i++) feed.request(lds, i);
            }
            if (landed > 0) landed--;
            else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(RA::WAIT) : "memory");
        }
        asm volatile("s_barrier" ::: "memory");
        if (fresh) feed.done();
    } else {
        if (!last) asm volatile("s_barrier" ::: "memory");     // of a tile: behind the epilogue
        feed.done();
    }
}

template <class T, int P, int ACT, bool Y32, int RES> __global__ __launch_bounds__(BIG_THREADS, 1) void linear_big_kernel(const Linear)
{
    using RA = Ring<P, true>;
    using RB = Ring<P, false>;
    static_assert(RA::N == RB::N && RA::PARTS <= 2, "");
    __shared__ __attribute__((aligned(128))) char lds[RA::N * RA::BYTES + RB::N * RB::BYTES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2;
    Feed<P> feed;
    feed.init(wave);
    const int ahead = half ? RB::AHEAD : RA::AHEAD;
#pragma unroll 1
    for (int i = 0; i < ahead; i++) feed.stage(lds);
    int landed = ahead - 1;                    // stages behind the current one that are known to be in LDS
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    uint32_t ci = blockIdx.x, slot_a = 0, slot_b = 0;
    if (half) asm volatile("s_barrier" ::: "memory");
    while (true) {
        f32x16 acc[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
        const BigItem now = big_item<P>(reload(), ci);
        const uint64_t count = now.count;
        const bool sum_rows = P == GWT && now.n0 == 0 && reload().colsum;
        float colsum = 0.f;
        const uint32_t steps = (uint32_t)((count + BIG_STEP - 1) / BIG_STEP);
        const int tail = (int)(count - (uint64_t)(steps - 1) * BIG_STEP);
        const bool odd = P != GWT && (tail & 7);
        const uint32_t whole = odd ? steps - 1 : steps;
        int sub = 0;
#pragma unroll 1
        for (uint32_t s = 0; s < whole; s++) {
            const bool fresh = sub == RA::PARTS - 1 || s + 1 == steps;
            big_step<T, P, false>(feed, acc, lds, slot_a, slot_b, sub, fresh, s + 1 == steps, wave, half, landed, 0, sum_rows, colsum);
            slot_b = slot_b + 1 == RB::N ? 0 : slot_b + 1;
            if (fresh) slot_a = slot_a + 1 == RA::N ? 0 : slot_a + 1;
            sub = fresh ? 0 : sub + 1;
        }
        if (odd) {
            big_step<T, P, true>(feed, acc, lds, slot_a, slot_b, sub, true, true, wave, half, landed, tail, false, colsum);
            slot_b = slot_b + 1 == RB::N ? 0 : slot_b + 1;
            slot_a = slot_a + 1 == RA::N ? 0 : slot_a + 1;
        }
        // the two halves' epilogues fall into the same change: half 0's behind its barrier, half 1's ahead of it
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        landed = ahead - 1;
        const Linear &g = reload();
        const BigItem c = big_item<P>(g, ci);
        if (P == GWT && sum_rows) {
            colsum += __shfl_xor(colsum, 32, WAVE);            // the two halves of each 16 k
            const uint32_t m = c.m0 + half * 128 + (wave & 3) * 32 + (threadIdx.x & 31);
            if ((threadIdx.x & 32) == 0 && m < g.M) g.colsum[c.split * g.M + m] = colsum;
        }
        epilogue<T, P, ACT, Y32, RES>(g, c, acc, half * 128, (wave & 3) * 64, P == GWT ? wave & 3 : 0);
        ci += g.blocks;
        if (ci >= g.items) break;
        if (half) asm volatile("s_barrier" ::: "memory");
    }
    // what was asked for behind the end was waited for above: nothing arrives in LDS that is another block's by then
}

// One kernel for each activation and width of the result: what a tile executes has to stay in the instruction cache.
template <class T> hipError_t launch_big(const Linear &g, int product, hipStream_t stream)
{
#define OPAL_BIG(P, ACT, Y32, RES)                                                                                          \
    if (product == P && (P == GWT || (g.act == ACT && (g.y_type == OPAL_F32) == Y32 && (!g.res ? 0 : g.res_type == OPAL_F32 ? RES32 : RES16) == RES))) {        \
        hipLaunchKernelGGL((linear_big_kernel<T, P, ACT, Y32, RES>), dim3(g.blocks), dim3(BIG_THREADS), 0, stream, g);       \
        return hipGetLastError();                                                                                           \
    }
#define OPAL_BIGS2(P, Y32, RES) \
    OPAL_BIG(P, ACT_NONE, Y32, RES) OPAL_BIG(P, ACT_RELU, Y32, RES) OPAL_BIG(P, ACT_SILU, Y32, RES) OPAL_BIG(P, ACT_GELU, Y32, RES)
#define OPAL_BIGS(P, Y32) OPAL_BIGS2(P, Y32, 0) OPAL_BIGS2(P, Y32, RES16) OPAL_BIGS2(P, Y32, RES32)
    OPAL_BIGS(FWD, false)
    OPAL_BIGS(FWD, true)
    OPAL_BIGS(GIN, false)
    OPAL_BIGS(GIN, true)
    OPAL_BIG(GWT, ACT_NONE, true, 0)
#undef OPAL_BIGS
#undef OPAL_BIGS2
#undef OPAL_BIG
    return hipErrorInvalidValue;
}

}  // namespace opal_head
