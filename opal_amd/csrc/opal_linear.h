// Matrix products of the score head: the tile kernel behind opal_linear, opal_linear_grad_input and opal_linear_grad_weight, and
// what its three translation units (one per element type) share.
//
//   C[m, n] = sum_k A(m, k) B(n, k), sums in 32 bits, then the epilogue of the product in question:
//     FWD  y  = act(x W^T + b) + r      A = x  [M, K], B = W [N, K]: the k of a row lie side by side in both ("KC")
//     GIN  dx = (dy W) act'(pre) + r    A = dy [M, K], B = W [K, N]: the n of a k lie side by side in W ("MC")
//     GWT  dW = dy^T x                  A = dy [K, M], B = x [K, N]: both MC, and K is the number of rows of the batch
//
// A block owns a BM x BN tile of C and walks k in steps of 128 bytes (64 elements of 16 bits, 32 of 32).  Both operands' tiles
// go to LDS as 16-byte chunks, twice buffered, and from there to registers as operands of v_mfma_f32_32x32x16 (16 bits) or
// v_mfma_f32_32x32x2_f32.  The MFMA's first operand is B and its second A, so a lane ends up with four neighbouring n of one m.
// 32-bit types: bound by the matrix pipe, 50 000 x 512 x 1564 (rows, N, K) 674 us, 119 TFLOP/s.  16-bit types: a step of 64 x 64 tiles is short against
// the way to memory, so what counts is that a CU has five blocks (four stages in LDS instead of two, for two blocks a CU, were slower):
// 16384 x 200 x 200 8 us; 100 000 x 128 x 1000 with 128 x 128 tiles 49 us, 525 TFLOP/s.
#pragma once
#include "opal_head.h"
#include "opal_linear_rules.h"

namespace opal_head {

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct Linear {
    const char *a, *b;
    uint64_t lda, ldb;            // row strides in elements
    uint64_t M, N, K;
    uint64_t ksplit;              // k handled by one block (a multiple of the step; >= K without a split)
    uint32_t tm, tn, splits;      // tiles along M and N, splits of K
    const float *bias;            // [N] or null
    const void *res; int res_type; uint64_t ldr;
    void *y; int y_type; uint64_t ldy;
    uint64_t y_split;             // elements between two splits' outputs
    const void *pre_in; void *pre_out; uint64_t ldp;   // the element type of the product
    int act;
    float *colsum;                // GWT: sums of dy's rows, [splits][M], by the tiles at n = 0; or null
    uint32_t few;                 // rows of a block of the kernel for few rows, in sixteens
    uint32_t items, blocks;       // tiles times splits, and the blocks that share them (opal_linear_big.h)
};

constexpr float GELU_A = 1.5957691216057308f, GELU_B = 0.044715f;   // 2 sqrt(2 / pi), and the cubic term of the tanh form

// v_exp_f32 and v_rcp_f32 are good to 1 ulp; the argument's rounding costs |z| 2^-24 of the result
constexpr float LOG2E = 1.44269504088896f;
__device__ __forceinline__ float sigmoid2(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z)); }      // of -z / LOG2E
__device__ __forceinline__ float gelu_sigmoid(float v) { return sigmoid2(v * (-LOG2E * GELU_A + -LOG2E * GELU_A * GELU_B * (v * v))); }
__device__ __forceinline__ float sigmoid(float z) { return sigmoid2(-LOG2E * z); }

__device__ __forceinline__ float act_value(float v, int act)
{
    if (act == ACT_RELU) return v > 0.f || v != v ? v : 0.f;
    if (act == ACT_SILU) return v * sigmoid(v);
    if (act == ACT_GELU) return v * gelu_sigmoid(v);
    return v;
}

__device__ __forceinline__ float act_slope(float v, int act)
{
    if (act == ACT_RELU) return v > 0.f ? 1.f : 0.f;      // NaN, whose result is NaN, passes nothing on
    const float c = fminf(fmaxf(v, -64.f), 64.f);      // beyond it p is 0 or 1 and c^2 p (1 - p) must not become 0 inf
    if (act == ACT_SILU) {
        const float p = sigmoid(v);
        return p + c * p * (1.f - p);
    }
    const float p = gelu_sigmoid(v);
    return p + c * p * (1.f - p) * GELU_A * (1.f + 3.f * GELU_B * c * c);
}

#ifdef __HIP_DEVICE_COMPILE__
#define OPAL_LDS __attribute__((address_space(3)))
#endif

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

// Where chunk c of row r of a KC tile lies within the row's eight: rows r and r + 1 share 256 bytes (all banks), the rotation by
// r >> 1 then spreads the same c of 16 rows over all 16 places, which is what a fragment read asks for.
__device__ __forceinline__ int swizzle_kc(int r) { return (r >> 1) & 7; }
// The same for the k-th line of an MC tile of R columns (in chunks).  16 bits: a transposing read takes 64 bytes of lines
// k .. k+3 and k+8 .. k+11; four lines get the four quarters of the banks (lines of 128 bytes: the two halves).
// 32 bits: a read takes 128 bytes of lines k and k + 4.
template <int ES, int R> __device__ __forceinline__ int swizzle_mc(int k)
{
    if constexpr (ES == 4) return ((k >> 2) & 1) << 3;
    else if constexpr (R * ES >= 256) return (k & 3) << 2;
    else return ((k >> 1) & 1) << 2;
}

// Transposing reads (ds_read_b64_tr_b16): 16 lanes read four lines of 16 columns, 8 bytes each, and get the four k of one column.
// Eight of them and their wait in one block: the builtin for this read makes the compiler wait for all chunks under way first.
// At a's and b's place (bytes) plus 0, H, K, K + H.
__device__ __forceinline__ uint32_t lds_place(const void *p)
{
#ifdef __HIP_DEVICE_COMPILE__
    return (uint32_t)(uintptr_t)(OPAL_LDS const void *)p;
#else
    return 0;
#endif
}
template <int H, int K> __device__ __forceinline__ void read_tr8(uint32_t a, uint32_t b, uint64_t (&x)[8])
{
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\t"
                 "ds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
                 "ds_read_b64_tr_b16 %2, %8 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %4, %9\n\t"
                 "ds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
                 "ds_read_b64_tr_b16 %6, %9 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                 : "v"(a), "v"(b), "n"(H), "n"(K), "n"(K + H)
                 : "memory");
#endif
}
__device__ __forceinline__ s16x8 join_tr(uint64_t lo, uint64_t hi)
{
    struct { uint64_t a, b; } v = {lo, hi};
    return __builtin_bit_cast(s16x8, v);
}

// where this lane's first transposing read of the 32 columns from r0 on begins, in an MC tile of R columns
template <int R> __device__ __forceinline__ uint32_t tr_place(int r0)
{
    const int lane = threadIdx.x & 63, col = r0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4, k = (lane >> 5) * 8 + ((lane >> 2) & 3);
    return (uint32_t)(k * (R * 2) + (((col >> 3) ^ swizzle_mc<2, R>(k)) * 16) + (col & 7) * 2);
}

// One operand's tile: R rows (m or n) of one step of k.
template <class T, int R, bool KC, int NT, bool DMA> struct Operand {
    static constexpr int ES = sizeof(T), EPC = 16 / ES, STEP = STEP_BYTES / ES;
    static constexpr int CHUNKS = R * 8, PER = CHUNKS / NT, LINE = KC ? 8 : R / EPC;   // LINE: chunks of a line
    static_assert(CHUNKS % NT == 0, "whole chunks per thread");
    const char *base;             // element (row r0, k0) of the matrix
    uint64_t ld;                  // bytes
    int rows;                     // of the tile, within the matrix
    u32x4 reg[DMA ? 1 : PER];

    __device__ __forceinline__ static int swz(int line) { return KC ? swizzle_kc(line) : swizzle_mc<ES, R>(line); }

    // Starts the loads of the step that begins at `base`, of which krem values of k are left.
    __device__ __forceinline__ void fetch(char *lds, uint64_t krem)
    {
        const int tid = threadIdx.x;
        const int kval = (int)(krem < (uint64_t)STEP ? krem : (uint64_t)STEP);
        if constexpr (DMA) {
#ifdef __HIP_DEVICE_COMPILE__
            // 16-byte aligned matrix and lines: whole chunks straight into LDS.  The buffer ends with the chunk that holds the
            // step's last element; lines behind it read as zeros.  A chunk that begins within the matrix lies whole in its
            // page; what it holds behind the matrix's edge is either never used (columns) or cleared by clear_tail (k).
            const uint32_t len = (uint32_t)((((uint64_t)(KC ? rows : kval) - 1) * ld + (uint64_t)(KC ? kval : rows) * ES + 15) & ~15ull);
            auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, (int)len, 0x00020000);
            const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int q = i * NT + tid, line = q / LINE, c = (q % LINE) ^ swz(line);
                uint32_t off = (uint32_t)line * (uint32_t)ld + (uint32_t)c * 16u;
                if (KC && c * EPC >= kval) off = 0x80000000u;      // behind every buffer (len < 2^31)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (OPAL_LDS void *)(lds + (i * NT + wave * WAVE) * 16), 16, (int)off, 0, 0, 0);
            }
#endif
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int q = i * NT + tid, line = q / LINE, c = (q % LINE) ^ swz(line);
                const int lines = KC ? rows : kval, width = KC ? kval : rows;
                const int left = width - c * EPC;
                const char *p = base + (uint64_t)line * ld + c * 16;
                u32x4 v = {0, 0, 0, 0};
                if (line < lines && left > 0) {
                    if (left >= EPC) {
                        struct __attribute__((packed, aligned(sizeof(T)))) Any { uint32_t w[4]; };
                        const Any a = *reinterpret_cast<const Any *>(p);
                        v = u32x4{a.w[0], a.w[1], a.w[2], a.w[3]};
                    } else {
                        if constexpr (ES == 4) {
#pragma unroll
                            for (int e = 0; e < EPC - 1; e++)
                                if (e < left) v[e] = ((const uint32_t *)p)[e];
                        } else {
#pragma unroll
                            for (int e = 0; e < EPC - 1; e++)
                                if (e < left) v[e / 2] |= (uint32_t)((const uint16_t *)p)[e] << (16 * (e & 1));
                        }
                    }
                }
                reg[i] = v;
            }
        }
    }
    __device__ __forceinline__ void commit(char *lds)
    {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < PER; i++) *reinterpret_cast<u32x4 *>(lds + (i * NT + threadIdx.x) * 16) = reg[i];
        }
    }
    __device__ __forceinline__ void advance() { base += KC ? (uint64_t)STEP_BYTES : (uint64_t)STEP * ld; }

    // The k behind the matrix's edge in the last chunk of each row (KC): whatever lies there must not meet a NaN-free sum.
    __device__ __forceinline__ static void clear_tail(char *lds, int kval)
    {
        if constexpr (KC && DMA) {
            const int keep = kval % EPC, c = kval / EPC;      // the chunk holds `keep` values of k; the caller checked keep != 0
            for (int r = threadIdx.x; r < R; r += NT) {
                T *p = reinterpret_cast<T *>(lds + r * STEP_BYTES + ((c ^ swizzle_kc(r)) * 16));
#pragma unroll
                for (int e = 1; e < EPC; e++)
                    if (e >= keep) p[e] = (T)0.f;
            }
        }
    }

    // Fragments of 32 rows from r0 on and a step's four times 16 k, 16-bit types: k = 16 kk + 8 (lane / 32) + 0..7 of row r0 + lane % 32.
    __device__ __forceinline__ static void frag16(const char *lds, int r0, s16x8 (&f)[4])
    {
        const int lane = threadIdx.x & 63;
        if constexpr (KC) {
            const int r = r0 + (lane & 31);
#pragma unroll
            for (int kk = 0; kk < 4; kk++) f[kk] = *reinterpret_cast<const s16x8 *>(lds + r * STEP_BYTES + (((kk * 2 + (lane >> 5)) ^ swizzle_kc(r)) * 16));
        } else {
            const uint32_t a = lds_place(lds) + tr_place<R>(r0);
            uint64_t x[8];
            read_tr8<4 * R * 2, 16 * R * 2>(a, a + 32 * R * 2, x);
#pragma unroll
            for (int kk = 0; kk < 4; kk++) f[kk] = join_tr(x[2 * kk], x[2 * kk + 1]);
        }
    }
    // 32-bit type: k = 8 j + 4 (lane / 32) + 0..3 of row r0 + lane % 32.
    __device__ __forceinline__ static f32x4 frag32(const char *lds, int r0, int j)
    {
        const int lane = threadIdx.x & 63, r = r0 + (lane & 31);
        if constexpr (KC) {
            const int c = j * 2 + (lane >> 5);
            return *reinterpret_cast<const f32x4 *>(lds + r * STEP_BYTES + ((c ^ swizzle_kc(r)) * 16));
        } else {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int k = j * 8 + (lane >> 5) * 4 + e;
                v[e] = *reinterpret_cast<const float *>(lds + k * (R * ES) + (((r >> 2) ^ swizzle_mc<ES, R>(k)) * 16) + (r & 3) * 4);
            }
            return v;
        }
    }
};

// the eight values of a fragment's lane, added up in 32 bits
template <class T> __device__ __forceinline__ float sum8(s16x8 f)
{
    struct V { T v[8]; };
    const V x = __builtin_bit_cast(V, f);
    return (((float)x.v[0] + (float)x.v[1]) + ((float)x.v[2] + (float)x.v[3])) + (((float)x.v[4] + (float)x.v[5]) + ((float)x.v[6] + (float)x.v[7]));
}

// The instruction adds float16 products without normalising subnormal operands first: a sum is rounded as if those were 2^-14 (measured: two products
// around 1e-6, one of them with an operand of 2^-18, off by 2^-42).
template <class T> __device__ __forceinline__ f32x16 mfma16(s16x8 a, s16x8 b, f32x16 c)
{
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (__is_same(T, bf16_t)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#else
    return c;
#endif
}

// Tile of a block.  Consecutive blocks go to the eight XCDs in turn, each with an L2 of its own; the tiles of an XCD are
// consecutive ones, the tiles along N of the same rows side by side, so that A's rows are read from HBM once per XCD.
__device__ __forceinline__ uint32_t xcd_tile(uint32_t b, uint32_t total)
{
    const uint32_t x = b & 7u, per = total >> 3, extra = total & 7u;
    return x * per + (x < extra ? x : extra) + (b >> 3);
}

// The epilogue of four neighbouring results of a row, `ncol` of them the matrix's
template <class T, int P> __device__ __forceinline__ void finish_quad(const Linear &g, f32x4 v, uint64_t m, uint64_t n, int ncol, f32x4 bias, uint64_t split)
{
    constexpr int own = __is_same(T, float) ? OPAL_F32 : __is_same(T, f16_t) ? OPAL_F16 : OPAL_BF16;
    if constexpr (P == FWD) {
        v += bias;
        if (g.pre_out) store4_typed(g.pre_out, own, m * g.ldp + n, ncol, v);
        if (g.act)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = act_value(v[e], g.act);
    }
    if constexpr (P == GIN) {
        if (g.act) {
            const f32x4 z = load4_typed(g.pre_in, own, m * g.ldp + n, ncol);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] *= act_slope(z[e], g.act);
        }
    }
    if (P != GWT && g.res) v += load4_typed(g.res, g.res_type, m * g.ldr + n, ncol);
    store4_typed(g.y, g.y_type, split * g.y_split + m * g.ldy + n, ncol, v);
}

template <class T, int P, int BM, int BN, int WM, int WN, bool DMA>
__global__ __launch_bounds__(WM * WN * WAVE) void linear_kernel(const Linear g)
{
    constexpr int NT = WM * WN * WAVE, ES = sizeof(T), STEP = STEP_BYTES / ES;
    constexpr int FM = BM / WM, FN = BN / WN, TM = FM / 32, TN = FN / 32;     // a wave's part and its fragments
    using OA = Operand<T, BM, P != GWT, NT, DMA>;
    using OB = Operand<T, BN, P == FWD, NT, DMA>;
    constexpr int STAGE = (BM + BN) * STEP_BYTES, EP_LD = FN + 4, EPI = WM * WN * 32 * EP_LD * 4;
    __shared__ __attribute__((aligned(128))) char lds[2 * STAGE > EPI ? 2 * STAGE : EPI];

    uint32_t t = xcd_tile(blockIdx.x, gridDim.x);
    const uint32_t tiles = g.tm * g.tn, split = t / tiles;
    t -= split * tiles;
    const uint64_t m0 = (uint64_t)(t / g.tn) * BM, n0 = (uint64_t)(t % g.tn) * BN;
    const uint64_t kbeg = split * g.ksplit, kend = kbeg + g.ksplit < g.K ? kbeg + g.ksplit : g.K;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = (wave / WN) * FM, wn = (wave % WN) * FN;

    OA A;
    OB B;
    A.ld = g.lda * ES;
    B.ld = g.ldb * ES;
    A.rows = (int)(g.M - m0 < (uint64_t)BM ? g.M - m0 : (uint64_t)BM);
    B.rows = (int)(g.N - n0 < (uint64_t)BN ? g.N - n0 : (uint64_t)BN);
    A.base = g.a + (P != GWT ? m0 * A.ld + kbeg * ES : kbeg * A.ld + m0 * ES);
    B.base = g.b + (P == FWD ? n0 * B.ld + kbeg * ES : kbeg * B.ld + n0 * ES);

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

    const bool sum_rows = P == GWT && n0 == 0 && wave % WN == 0 && g.colsum;      // one wave for each block of rows
    float colsum[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) colsum[i] = 0.f;
    uint64_t krem = kend - kbeg;
    char *cur = lds, *nxt = lds + STAGE;
    if (krem) {
        A.fetch(cur, krem);
        B.fetch(cur + BM * STEP_BYTES, krem);
        A.commit(cur);
        B.commit(cur + BM * STEP_BYTES);
    }
    while (krem) {
        __syncthreads();          // the step's chunks are in LDS, and nobody reads the other half any more
        const bool more = krem > (uint64_t)STEP;
        if (more) {
            A.advance();
            B.advance();
            A.fetch(nxt, krem - STEP);
            B.fetch(nxt + BM * STEP_BYTES, krem - STEP);
        } else if (DMA && P != GWT && krem % OA::EPC) {
            OA::clear_tail(cur, (int)krem);
            OB::clear_tail(cur + BM * STEP_BYTES, (int)krem);
            __syncthreads();
        }
        const char *la = cur, *lb = cur + BM * STEP_BYTES;
        if constexpr (ES == 2) {
            s16x8 fa[TM][4], fb[TN][4];
#pragma unroll
            for (int i = 0; i < TM; i++) OA::frag16(la, wm + i * 32, fa[i]);
#pragma unroll
            for (int j = 0; j < TN; j++) OB::frag16(lb, wn + j * 32, fb[j]);
            if (P == GWT && sum_rows) {
#pragma unroll
                for (int i = 0; i < TM; i++)
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) colsum[i] += sum8<T>(fa[i][kk]);
            }
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
#pragma unroll
                for (int i = 0; i < TM; i++)
#pragma unroll
                    for (int j = 0; j < TN; j++) acc[i][j] = mfma16<T>(fb[j][kk], fa[i][kk], acc[i][j]);
        } else {
#pragma unroll
            for (int kk = 0; kk < STEP / 8; kk++) {
                f32x4 fa[TM], fb[TN];
#pragma unroll
                for (int i = 0; i < TM; i++) fa[i] = OA::frag32(la, wm + i * 32, kk);
#pragma unroll
                for (int j = 0; j < TN; j++) fb[j] = OB::frag32(lb, wn + j * 32, kk);
                if (P == GWT && sum_rows)
#pragma unroll
                    for (int i = 0; i < TM; i++) colsum[i] += (fa[i][0] + fa[i][1]) + (fa[i][2] + fa[i][3]);
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int i = 0; i < TM; i++)
#pragma unroll
                        for (int j = 0; j < TN; j++) {
#ifdef __HIP_DEVICE_COMPILE__
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j][e], fa[i][e], acc[i][j], 0, 0, 0);
#endif
                        }
            }
        }
        if (more) {
            A.commit(nxt);
            B.commit(nxt + BM * STEP_BYTES);
        }
        char *const s = cur;
        cur = nxt;
        nxt = s;
        krem = more ? krem - STEP : 0;
    }

    if (P == GWT && sum_rows) {
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const float s = colsum[i] + __shfl_xor(colsum[i], 32, WAVE);      // lanes l and l + 32 held the row's halves of k
            const uint64_t m = m0 + wm + i * 32 + (lane & 31);
            if (lane < 32 && m < g.M) g.colsum[split * g.M + m] = s;
        }
    }

    // Epilogue: each wave turns 32 rows at a time in its own part of the LDS, so that neighbouring lanes hold neighbouring
    // columns of a row when the residual and the pre-activation are read and the results written.
    __syncthreads();
    float *turn = reinterpret_cast<float *>(lds) + wave * 32 * EP_LD;
    constexpr int LPR = FN / 4, RPP = WAVE / LPR;          // lanes per row, rows per pass
    const int col = (lane % LPR) * 4;
    const uint64_t n = n0 + wn + col;
    const int ncol = n < g.N ? (int)(g.N - n < 4 ? g.N - n : 4) : 0;
    f32x4 bias = {0.f, 0.f, 0.f, 0.f};
    if (P == FWD && g.bias && ncol) bias = load4_typed(g.bias, OPAL_F32, n, ncol);
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<f32x4 *>(turn + (lane & 31) * EP_LD + j * 32 + q * 8 + (lane >> 5) * 4) =
                    f32x4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
        wave_order();
        for (int p = 0; p < 32 / RPP; p++) {
            const int r = p * RPP + lane / LPR;
            const uint64_t m = m0 + wm + i * 32 + r;
            f32x4 v = *reinterpret_cast<const f32x4 *>(turn + r * EP_LD + col);
            if (m >= g.M || !ncol) continue;
            finish_quad<T, P>(g, v, m, n, ncol, bias, split);
        }
        wave_order();
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// FWD and GIN with few rows: reading W once is all there is to do, and what counts is that all of the card asks for it at once.  A
// block takes 16 columns and 16 TM rows; its eight waves share the k between them, 32 (16 for 32-bit types) at a time, operands straight from
// memory to v_mfma_f32_16x16x32 / 16x16x4_f32, and add up in LDS.  No LDS on the way in, no barrier but one.  One row of 1564 x 512 in
// bfloat16: 4.7 us, of which the launch is most.
constexpr int FEW_WAVES = 8;

// A fragment's lane: EPC values of k from k0 on of line r (KC), or column r of lines k0 .. (MC); beyond the matrix: zeros
template <class T, bool KC> __device__ __forceinline__ u32x4 lane_k(const T *p, uint64_t ld, uint64_t r, bool in, uint64_t k0, uint64_t K)
{
    constexpr int EPC = 16 / sizeof(T);
    u32x4 v = {0, 0, 0, 0};
    if (!in || k0 >= K) return v;
    const int left = K - k0 < (uint64_t)EPC ? (int)(K - k0) : EPC;
    if (KC && left == EPC) {
        typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));     // (a vector: a struct's 32-bit words would be loaded one by one)
        return *reinterpret_cast<const Any *>(p + r * ld + k0);
    }
#pragma unroll
    for (int e = 0; e < EPC; e++)
        if (e < left) {
            const T *q = KC ? p + r * ld + k0 + e : p + (k0 + e) * ld + r;
            if constexpr (sizeof(T) == 4) v[e] = *reinterpret_cast<const uint32_t *>(q);
            else v[e / 2] |= (uint32_t)*reinterpret_cast<const uint16_t *>(q) << (16 * (e & 1));
        }
    return v;
}

template <class T> __device__ __forceinline__ f32x4 mfma_few(u32x4 a, u32x4 b, f32x4 c)
{
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (__is_same(T, bf16_t)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (__is_same(T, f16_t)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
#else
    return c;
#endif
}

template <class T, int P, int TM> __global__ __launch_bounds__(FEW_WAVES * WAVE) void linear_few_kernel(const Linear g)
{
    constexpr int EPC = 16 / sizeof(T), STEP = 4 * EPC, U = TM == 1 ? 8 : 4;
    __shared__ f32x4 red[FEW_WAVES][TM][WAVE];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r16 = lane & 15, kq = (lane >> 4) * EPC;
    const uint64_t n0 = (uint64_t)(blockIdx.x % g.tn) * 16, m0 = (uint64_t)(blockIdx.x / g.tn) * (16 * TM);
    const T *A = (const T *)g.a, *B = (const T *)g.b;
    f32x4 acc[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint64_t k = (uint64_t)wave * STEP; k < g.K; k += (uint64_t)U * FEW_WAVES * STEP) {
        u32x4 b[U], a[U][TM];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t ku = k + (uint64_t)u * FEW_WAVES * STEP + kq;
            b[u] = lane_k<T, P == FWD>(B, g.ldb, n0 + r16, n0 + r16 < g.N, ku, g.K);
#pragma unroll
            for (int i = 0; i < TM; i++) a[u][i] = lane_k<T, true>(A, g.lda, m0 + i * 16 + r16, m0 + i * 16 + r16 < g.M, ku, g.K);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < TM; i++) acc[i] = mfma_few<T>(b[u], a[u][i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < TM; i++) red[wave][i][lane] = acc[i];
    __syncthreads();
    if (threadIdx.x >= TM * WAVE) return;
    f32x4 v = red[0][wave][lane];
#pragma unroll
    for (int w = 1; w < FEW_WAVES; w++) v += red[w][wave][lane];
    const uint64_t m = m0 + wave * 16 + r16, n = n0 + (lane >> 4) * 4;           // four columns of a row
    if (m >= g.M || n >= g.N) return;
    const int ncol = g.N - n < 4 ? (int)(g.N - n) : 4;
    finish_quad<T, P>(g, v, m, n, ncol, P == FWD && g.bias ? load4_typed(g.bias, OPAL_F32, n, ncol) : f32x4{0.f, 0.f, 0.f, 0.f}, 0);
}

// GWT of few rows: a block takes 32 x 32 results over all rows, which its sixteen waves share between them, and adds up in LDS: one launch
// and no workspace, where splits would need a second launch to add them up.  Operands come straight from memory, all of a wave's
// loads for 64 rows (32 of 32-bit types) at once.  16 bits: a lane loads two neighbouring columns of eight rows; its even ones are one operand of
// v_mfma_f32_16x16x32, its odd ones another.
constexpr int FEWW_WAVES = 16, FEWW_LD = 33;

template <class T> struct FewCols {            // a lane's loads of one operand
    static constexpr bool W16 = sizeof(T) == 2;
    static constexpr int ROWS = W16 ? 8 : 1, PER = W16 ? 32 : 4, NV = W16 ? 8 : 2;      // rows of a lane and of a wave, registers
    const char *p;
    uint64_t ld;                               // (the same for all lanes, as p)
    uint32_t off, more;                        // more: 32 bits: the other 16 columns are the next ones, or these again
    int row;                                   // this lane's first row
    bool edge;                                 // 16 bits: the second column is behind the matrix's edge
    // columns c0 .. c0 + 31 of `cols`; lanes behind the edge read its last ones (whose results nobody writes)
    __device__ __forceinline__ void init(const char *base, uint64_t stride, uint32_t c0, uint32_t cols, int lane)
    {
        uint32_t c = c0 + (W16 ? 2 : 1) * (lane & 15);
        if (c >= cols) c = W16 ? (cols - 1) & ~1u : cols - 1;
        ld = stride * sizeof(T);
        p = base;
        row = (lane >> 4) * ROWS;
        off = (uint32_t)row * (uint32_t)ld + c * sizeof(T);          // less than 2^28: 24 rows of 2^22 bytes
        more = c + 16 < cols ? 64 : 0;
        edge = W16 && c + 1 == cols;
    }
    // This lane's rows of those from k on; CUT: those from `end` on as zeros, and nothing behind the edge (which, in all rows but the
    // matrix's last, is the next element in memory: read with its neighbour, used by no result).
    template <bool CUT> __device__ __forceinline__ void load(uint64_t k, uint64_t end, uint32_t (&v)[NV]) const
    {
        struct __attribute__((packed, aligned(2))) Any { uint32_t w; };
#pragma unroll
        for (int e = 0; e < NV; e++) {
            const uint64_t r = k + (W16 ? e : 0);
            v[e] = 0;
            if (CUT && r + row >= end) continue;
            const char *q = p + r * ld + (off + (W16 ? 0 : e * more));
            if (CUT && edge) v[e] = *reinterpret_cast<const uint16_t *>(q);
            else v[e] = reinterpret_cast<const Any *>(q)->w;
        }
    }
};

template <class T> __global__ __launch_bounds__(FEWW_WAVES * WAVE) void linear_few_weight_kernel(const Linear g)
{
    using C = FewCols<T>;
    constexpr bool W16 = C::W16;
    constexpr int NV = C::NV, U = W16 ? 2 : 8;
    __shared__ float red[FEWW_WAVES][32 * FEWW_LD];
    __shared__ float sums[FEWW_WAVES * 4][32];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c16 = lane & 15;
    const uint32_t n0 = (blockIdx.x % g.tn) * 32, m0 = (blockIdx.x / g.tn) * 32;
    C a, b;
    a.init(g.a, g.lda, m0, (uint32_t)g.M, lane);
    b.init(g.b, g.ldb, n0, (uint32_t)g.N, lane);
    const bool sum_rows = n0 == 0 && g.colsum;
    f32x4 acc[2][2];                           // [n][m]: even and odd columns (16 bits), the first and the second sixteen
#pragma unroll
    for (int i = 0; i < 2; i++) acc[i][0] = acc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    float cs[2] = {0.f, 0.f};
    auto use = [&](const uint32_t (&va)[NV], const uint32_t (&vb)[NV]) __attribute__((always_inline)) {
        u32x4 fa[2], fb[2];
        if constexpr (W16) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                fa[0][i] = __builtin_amdgcn_perm(va[2 * i + 1], va[2 * i], 0x05040100);
                fa[1][i] = __builtin_amdgcn_perm(va[2 * i + 1], va[2 * i], 0x07060302);
                fb[0][i] = __builtin_amdgcn_perm(vb[2 * i + 1], vb[2 * i], 0x05040100);
                fb[1][i] = __builtin_amdgcn_perm(vb[2 * i + 1], vb[2 * i], 0x07060302);
            }
            if (sum_rows) {
                cs[0] += sum8<T>(__builtin_bit_cast(s16x8, fa[0]));
                cs[1] += sum8<T>(__builtin_bit_cast(s16x8, fa[1]));
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = mfma_few<T>(fb[i], fa[j], acc[i][j]);
        } else {
            const float x0 = __builtin_bit_cast(float, va[0]), x1 = __builtin_bit_cast(float, va[1]), y0 = __builtin_bit_cast(float, vb[0]), y1 = __builtin_bit_cast(float, vb[1]);
            if (sum_rows) {
                cs[0] += x0;
                cs[1] += x1;
            }
#ifdef __HIP_DEVICE_COMPILE__
            acc[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(y0, x0, acc[0][0], 0, 0, 0);
            acc[0][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(y0, x1, acc[0][1], 0, 0, 0);
            acc[1][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(y1, x0, acc[1][0], 0, 0, 0);
            acc[1][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(y1, x1, acc[1][1], 0, 0, 0);
#endif
        }
    };
    uint64_t k = (uint64_t)wave * (U * C::PER);
    for (; k + U * C::PER < g.K; k += (uint64_t)FEWW_WAVES * U * C::PER) {
        uint32_t va[U][NV], vb[U][NV];
#pragma unroll
        for (int u = 0; u < U; u++) {
            a.template load<false>(k + u * C::PER, 0, va[u]);
            b.template load<false>(k + u * C::PER, 0, vb[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) use(va[u], vb[u]);
    }
    for (uint64_t end = k + U * C::PER < g.K ? k + U * C::PER : g.K; k < end; k += C::PER) {      // the rows up to the last one, one wave's
        uint32_t va[NV], vb[NV];
        a.template load<true>(k, g.K, va);
        b.template load<true>(k, g.K, vb);
        use(va, vb);
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int n = (lane >> 4) * 4 + r;
                red[wave][(W16 ? 2 * c16 + j : j * 16 + c16) * FEWW_LD + (W16 ? 2 * n + i : i * 16 + n)] = acc[i][j][r];
            }
    if (sum_rows)
#pragma unroll
        for (int j = 0; j < 2; j++) sums[wave * 4 + (lane >> 4)][W16 ? 2 * c16 + j : j * 16 + c16] = cs[j];
    __syncthreads();
    const uint32_t r = threadIdx.x >> 5, c = threadIdx.x & 31;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < FEWW_WAVES; w++) v += red[w][r * FEWW_LD + c];
    if (m0 + r < g.M && n0 + c < g.N) ((float *)g.y)[(uint64_t)(m0 + r) * g.ldy + n0 + c] = v;
    if (sum_rows && threadIdx.x < 32 && m0 + c < g.M) {
        v = 0.f;
#pragma unroll 8
        for (int w = 0; w < FEWW_WAVES * 4; w++) v += sums[w][c];
        g.colsum[m0 + c] = v;
    }
}

// The launch of one product in one element type (opal_linear_{f32,f16,bf16}.hip); tile: opal_linear_rules.h.
template <class T> hipError_t launch_linear(const Linear &g, int product, int tile, bool dma, hipStream_t stream);

#define OPAL_LINEAR_CASE(T, P, TILE, BM, BN, WM, WN, D)                                                                              \
    if (product == P && tile == TILE && dma == D) {                                                                                  \
        hipLaunchKernelGGL((linear_kernel<T, P, BM, BN, WM, WN, D>), dim3(g.tm * g.tn * g.splits), dim3(WM * WN * WAVE), 0, stream, g); \
        return hipGetLastError();                                                                                                    \
    }
#define OPAL_LINEAR_FEW(T, P, TM)                                                                                                   \
    if (product == P && tile == 3 && g.few == TM) {                                                                                  \
        hipLaunchKernelGGL((linear_few_kernel<T, P, TM>), dim3(g.tm * g.tn), dim3(FEW_WAVES * WAVE), 0, stream, g);                   \
        return hipGetLastError();                                                                                                    \
    }
#define OPAL_LINEAR_FEW_WEIGHT(T)                                                                                                   \
    if (product == GWT && tile == 5) {                                                                                               \
        hipLaunchKernelGGL((linear_few_weight_kernel<T>), dim3(g.tm * g.tn), dim3(FEWW_WAVES * WAVE), 0, stream, g);                  \
        return hipGetLastError();                                                                                                    \
    }
#define OPAL_LINEAR_SMALL(T, P)                       \
    OPAL_LINEAR_CASE(T, P, 0, 64, 64, 2, 2, true)     \
    OPAL_LINEAR_CASE(T, P, 0, 64, 64, 2, 2, false)
#define OPAL_LINEAR_CASES(T, P)                       \
    OPAL_LINEAR_SMALL(T, P)                           \
    OPAL_LINEAR_CASE(T, P, 1, 128, 128, 2, 2, true)   \
    OPAL_LINEAR_CASE(T, P, 1, 128, 128, 2, 2, false)

}  // namespace opal_head
