// Row operators of the score head: layer norm (forward, backward with the reduction of the weight's gradient) and the softmax loss
// over the class scores; and the C entry points of these and of the matrix products (opal_linear.h).
//
//   layer norm   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), y = (x - m) r g + b
//   backward     h = dy g, xh = (x - m) r:  dx = r (h - mean(h) - xh mean(h xh));  dg = sum_rows dy xh,  db = sum_rows dy
//   softmax      e_j = exp(s_j - max), Z = sum e_j:  loss = log Z + max - s_label, grad_j = scale (e_j / Z - [j is the label])
//
// A row belongs to a team of 16, 32 or 64 lanes (up to 128, 512, 2048 columns), which holds it in registers: one read of memory, sums
// over the team's lanes; up to 8192 columns to a block of 256 threads in the same way; a longer one is read again by a block of
// 1024 for each pass.
#include <algorithm>
#include <cmath>
#include <string>

#include "opal_linear.h"

namespace opal_head {

constexpr int BLOCK = 256;

// Sums and maxima over the TPR threads of a row: 16, 32 or 64 lanes, or the whole block (red: one float per wave and value, two
// buffers in turn so that a block needs one barrier per reduction).
template <int TPR> struct Team {
    float *red;
    int turn = 0;
    __device__ __forceinline__ float join(float v, bool take_max)
    {
        if constexpr (TPR <= WAVE) return take_max ? wave_max<TPR>(v) : wave_sum<TPR>(v);
        else {
            v = take_max ? wave_max(v) : wave_sum(v);
            constexpr int NW = TPR / WAVE;
            float *r = red + (turn ^= NW);
            if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
            __syncthreads();
            float t = r[0];
            for (int i = 1; i < NW; i++) t = take_max ? fmaxf(t, r[i]) : t + r[i];
            return t;
        }
    }
    __device__ __forceinline__ float sum(float v) { return join(v, false); }
    __device__ __forceinline__ float max(float v) { return join(v, true); }
};

// A thread's share of a row: quads i * TPR + t, i < NQ.  Teams within a wave have NQ = ceil(cols / (4 TPR)): all quads but the last are whole.
template <int TPR, int NQ> __device__ __forceinline__ int quad_col(int i, int t) { return (i * TPR + t) * 4; }
template <int TPR, int NQ> __device__ __forceinline__ int quad_left(int i, int col, int cols)
{
    return TPR <= WAVE && i < NQ - 1 ? 4 : cols - col;
}

template <class T> constexpr int type_of() { return __is_same(T, float) ? OPAL_F32 : __is_same(T, f16_t) ? OPAL_F16 : OPAL_BF16; }

template <class T, int TPR, int NQ>
__device__ __forceinline__ void load_row(const T *row, int t, int cols, float fill, f32x4 (&v)[NQ])
{
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int col = quad_col<TPR, NQ>(i, t);
        v[i] = load4_typed(row, type_of<T>(), col, quad_left<TPR, NQ>(i, col, cols), fill);
    }
}

struct Norm {
    const void *x; uint64_t ldx;
    const float *gamma, *beta;
    uint64_t n; int cols; float eps;
    void *y; int y_type; uint64_t ldy;
    float *mean, *rstd;
    uint64_t first;                            // row of the launch's first block
};

__device__ __forceinline__ f32x4 param4(const float *p, int col, int left, float none)
{
    return p ? load4_typed(p, OPAL_F32, col, left, none) : f32x4{none, none, none, none};
}

// Bound by memory: 250 000 x 1564 float32 -> bfloat16 414 us, 5.7 TB/s (a plain conversion of the same matrix: 5.8).
template <class T, int TPR, int NQ, bool NT> __global__ __launch_bounds__(BLOCK) void norm_kernel(const Norm g)
{
    __shared__ float red[2 * BLOCK / WAVE];
    Team<TPR> team{red};
    constexpr int RPB = BLOCK / TPR;
    const int t = threadIdx.x % TPR;
    const float cols = (float)g.cols;
    const uint64_t row = g.first + (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row >= g.n) return;
    f32x4 x[NQ];
    load_row<T, TPR, NQ>((const T *)g.x + row * g.ldx, t, g.cols, 0.f, x);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; i++) s += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
    const float mean = team.sum(s) / cols;      // a division: the mean of equal values is that value
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[i][e] -= mean;
            if (quad_left<TPR, NQ>(i, quad_col<TPR, NQ>(i, t), g.cols) > e) s += x[i][e] * x[i][e];
        }
    const float rstd = 1.f / sqrtf(team.sum(s) / cols + g.eps);
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int col = quad_col<TPR, NQ>(i, t), left = quad_left<TPR, NQ>(i, col, g.cols);
        const f32x4 ga = param4(g.gamma, col, left, 1.f), be = param4(g.beta, col, left, 0.f);
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = x[i][e] * rstd * ga[e] + be[e];
        store4_typed<NT>(g.y, g.y_type, row * g.ldy + col, left, y);
    }
    if (t == 0) {
        if (g.mean) g.mean[row] = mean;
        if (g.rstd) g.rstd[row] = rstd;
    }
}

constexpr int LONG = 1024;                // threads on a row that does not fit the registers: read again for each pass, mostly from the caches
                                          // (20 000 x 20 000 float32 -> bfloat16 1.1 ms, 2.2 TB/s of what it has to read and write)

template <class T> __global__ __launch_bounds__(LONG) void norm_long_kernel(const Norm g)
{
    __shared__ float red[2 * LONG / WAVE];
    Team<LONG> team{red};
    const float cols = (float)g.cols;
    for (uint64_t row = blockIdx.x; row < g.n; row += gridDim.x) {
        const T *x = (const T *)g.x + row * g.ldx;
        float s = 0.f;
        for (int c = threadIdx.x; c < g.cols; c += LONG) s += (float)x[c];
        const float mean = team.sum(s) / cols;      // a division: the mean of equal values is that value
        s = 0.f;
        for (int c = threadIdx.x; c < g.cols; c += LONG) { const float d = (float)x[c] - mean; s += d * d; }
        const float rstd = 1.f / sqrtf(team.sum(s) / cols + g.eps);
        for (int c = threadIdx.x; c < g.cols; c += LONG) {       // y may be x: a thread overwrites only what it alone reads
            const float y = ((float)x[c] - mean) * rstd * (g.gamma ? g.gamma[c] : 1.f) + (g.beta ? g.beta[c] : 0.f);
            store4_typed(g.y, g.y_type, row * g.ldy + c, 1, f32x4{y, 0.f, 0.f, 0.f});
        }
        if (threadIdx.x == 0) {
            if (g.mean) g.mean[row] = mean;
            if (g.rstd) g.rstd[row] = rstd;
        }
    }
}

struct NormBack {
    const void *dy; uint64_t lddy;
    const void *x; uint64_t ldx;
    const float *gamma, *mean, *rstd;
    uint64_t n; int cols;
    void *dx; int dx_type; uint64_t lddx;      // dx may be null
    float *part;                               // [blocks][2][cols]: dgamma, dbeta; null: not wanted, or one block's
    float *dgamma, *dbeta;                     // of one block, either may be null
    bool stream;                               // dx past the caches (stream_out)
};

// Threads of a block of the backward pass.  Short rows leave few bytes under way in a wave, so many waves share a block (and its one
// partial sum); long ones fill a wave's registers.
constexpr int back_threads(int TPR, int NQ) { return TPR > WAVE ? BLOCK : TPR * NQ <= 128 ? 1024 : TPR * NQ <= 256 ? 512 : BLOCK; }

// Every thread keeps the sums of its own columns over the rows that its team visits; the teams of a block add theirs up in
// order, and sum_parts_kernel adds the blocks': no atomics, the same bits every time.  The next row is asked for before the
// present one is worked on.  Bound by memory: 500 009 x 355 (float32 x and dx, bfloat16 dy) 354 us, 5.0 TB/s, of which the sums' 4.7.
template <class TX, class TY, int TPR, int NQ> __global__ __launch_bounds__(back_threads(TPR, NQ)) void norm_back_kernel(const NormBack g)
{
    constexpr int THREADS = back_threads(TPR, NQ), RPB = THREADS / TPR, WAVES = THREADS / WAVE;
    __shared__ float red[2 * BLOCK / WAVE];
    __shared__ f32x4 both[TPR <= WAVE ? 2 * NQ * TPR : 1];
    Team<TPR> team{red};
    const int t = threadIdx.x % TPR;
    const float cols = (float)g.cols;
    const uint64_t step = (uint64_t)gridDim.x * RPB;
    f32x4 dg[NQ], db[NQ];
#pragma unroll
    for (int i = 0; i < NQ; i++) dg[i] = db[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    RawOf<TX> xr[NQ];
    RawOf<TY> hr[NQ];
    float mean_next = 0.f, rstd_next = 0.f;
    auto ask = [&](uint64_t r) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int col = quad_col<TPR, NQ>(i, t), left = quad_left<TPR, NQ>(i, col, g.cols);
            xr[i] = load_raw_of((const TX *)g.x + r * g.ldx + col, left);
            hr[i] = load_raw_of((const TY *)g.dy + r * g.lddy + col, left);
        }
        mean_next = g.mean[r];
        rstd_next = g.rstd[r];
    };
    if (row < g.n) ask(row);
    for (; row < g.n; row += step) {
        f32x4 x[NQ], h[NQ];
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            x[i] = decode_of(xr[i]);
            h[i] = decode_of(hr[i]);
        }
        const float mean = mean_next, rstd = rstd_next;
        // in place (dx over x or dy) other rows than this one are not touched: the next one may be read before this is written
        if (row + step < g.n) ask(row + step);
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int col = quad_col<TPR, NQ>(i, t), left = quad_left<TPR, NQ>(i, col, g.cols);
            const f32x4 ga = param4(g.gamma, col, left, 1.f);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[i][e] = left > e ? (x[i][e] - mean) * rstd : 0.f;
                dg[i][e] += h[i][e] * x[i][e];
                db[i][e] += h[i][e];
                h[i][e] = left > e ? h[i][e] * ga[e] : 0.f;
                s0 += h[i][e];
                s1 += h[i][e] * x[i][e];
            }
        }
        if (!g.dx) continue;
        s0 = team.sum(s0) / cols;
        s1 = team.sum(s1) / cols;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int col = quad_col<TPR, NQ>(i, t), left = quad_left<TPR, NQ>(i, col, g.cols);
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = rstd * (h[i][e] - s0 - x[i][e] * s1);
            if (g.stream) store4_typed<true>(g.dx, g.dx_type, row * g.lddx + col, left, d);
            else store4_typed<false>(g.dx, g.dx_type, row * g.lddx + col, left, d);
        }
    }
    if (!g.part && !g.dgamma && !g.dbeta) return;
    if constexpr (TPR <= WAVE) {
#pragma unroll
        for (int i = 0; i < NQ; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {                      // a wave's teams
                if constexpr (TPR <= 16) {
                    dg[i][e] = add_exchanged<16>(dg[i][e]);
                    db[i][e] = add_exchanged<16>(db[i][e]);
                }
                if constexpr (TPR <= 32) {
                    dg[i][e] = add_exchanged<32>(dg[i][e]);
                    db[i][e] = add_exchanged<32>(db[i][e]);
                }
            }
        const bool first = (threadIdx.x & 63) < TPR;           // a team of each wave
        for (int w = 0; w < WAVES; w++) {
            if ((int)(threadIdx.x / WAVE) == w && first) {
#pragma unroll
                for (int i = 0; i < NQ; i++) {
                    f32x4 *a = both + i * TPR + t, *b = both + (NQ + i) * TPR + t;
                    if (w) {
                        dg[i] += *a;
                        db[i] += *b;
                    }
                    *a = dg[i];
                    *b = db[i];
                }
            }
            __syncthreads();
        }
        if ((int)(threadIdx.x / WAVE) != WAVES - 1 || !first) return;      // the last wave's team holds the block's sums
    }
    float *out = g.part + (uint64_t)blockIdx.x * 2 * g.cols;
    float *const to_dg = g.part ? out : g.dgamma, *const to_db = g.part ? out + g.cols : g.dbeta;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int col = quad_col<TPR, NQ>(i, t), left = quad_left<TPR, NQ>(i, col, g.cols);
        if (to_dg) store4_typed(to_dg, OPAL_F32, col, left, dg[i]);
        if (to_db) store4_typed(to_db, OPAL_F32, col, left, db[i]);
    }
}

template <class TX, class TY> __global__ __launch_bounds__(LONG) void norm_back_long_kernel(const NormBack g)
{
    __shared__ float red[2 * LONG / WAVE];
    Team<LONG> team{red};
    const float cols = (float)g.cols;
    for (uint64_t row = blockIdx.x; row < g.n; row += gridDim.x) {
        const TX *x = (const TX *)g.x + row * g.ldx;
        const TY *dy = (const TY *)g.dy + row * g.lddy;
        const float mean = g.mean[row], rstd = g.rstd[row];
        float s0 = 0.f, s1 = 0.f;
        for (int c = threadIdx.x; c < g.cols; c += LONG) {
            const float h = (float)dy[c] * (g.gamma ? g.gamma[c] : 1.f);
            s0 += h;
            s1 += h * (((float)x[c] - mean) * rstd);
        }
        s0 = team.sum(s0) / cols;
        s1 = team.sum(s1) / cols;
        for (int c = threadIdx.x; c < g.cols; c += LONG) {       // dx may be dy or x
            const float h = (float)dy[c] * (g.gamma ? g.gamma[c] : 1.f), xh = ((float)x[c] - mean) * rstd;
            store4_typed(g.dx, g.dx_type, row * g.lddx + c, 1, f32x4{rstd * (h - s0 - xh * s1), 0.f, 0.f, 0.f});
        }
    }
}

// The column sums of long rows: a block takes 256 columns of a run of rows.  Runs before the rows are overwritten by dx.
template <class TX, class TY> __global__ __launch_bounds__(BLOCK) void norm_cols_kernel(const NormBack g, uint64_t rows)
{
    const int c = blockIdx.x * BLOCK + threadIdx.x;
    if (c >= g.cols) return;
    const uint64_t beg = blockIdx.y * rows, end = beg + rows < g.n ? beg + rows : g.n;
    float dg = 0.f, db = 0.f;
    for (uint64_t r = beg; r < end; r++) {
        const float d = (float)((const TY *)g.dy)[r * g.lddy + c];
        dg += d * (((float)((const TX *)g.x)[r * g.ldx + c] - g.mean[r]) * g.rstd[r]);
        db += d;
    }
    float *out = g.part + (uint64_t)blockIdx.y * 2 * g.cols;
    out[c] = dg;
    out[(uint64_t)g.cols + c] = db;
}

// The sums over `parts` of [2][cols]: the first goes to out0, the second to out1 (either may be null), in a fixed order; parts == 0
// writes zeros.  A block takes 16 columns with 64 groups of parts.
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float *part, uint32_t parts, uint32_t cols, float *out0, float *out1)
{
    __shared__ float acc[64][16];
    const uint32_t c = threadIdx.x & 15, w = threadIdx.x >> 4;
    const uint64_t col = (uint64_t)blockIdx.x * 16 + c, width = 2ull * cols;
    float s = 0.f;
    if (col < width) {
#pragma unroll 8
        for (uint32_t p = w; p < parts; p += 64) s += part[p * width + col];
    }
    acc[w][c] = s;
    __syncthreads();
    for (uint32_t half = 32; half; half >>= 1) {
        if (w < half) acc[w][c] += acc[w + half][c];
        __syncthreads();
    }
    if (w == 0 && col < width) {
        float *out = col < cols ? out0 : out1;
        if (out) out[col < cols ? col : col - cols] = acc[0][c];
    }
}

// ------------------------------------------------------------------------------------------------ softmax
struct Softmax {
    const void *s; uint64_t lds;
    uint64_t n; int cols;
    const int32_t *labels; float scale;
    float *loss;
    void *grad; int grad_type; uint64_t ldg;
    int32_t *out_class; float *out_prob;
    unsigned long long *bad;
    uint64_t first;                            // row of the launch's first block
};

// What is known of a row once its maximum and the sum of exponentials are: written by one thread.
__device__ __forceinline__ void softmax_row(const Softmax &g, uint64_t row, float top, float total, int best, int label, bool bad, float at_label)
{
    if (bad) atomicAdd(g.bad, 1ull);
    // a row of nothing but -inf has no class with a probability: total is 0
    if (g.loss) g.loss[row] = label < 0 ? 0.f : total == 0.f ? INFINITY : logf(total) + (top - at_label);
    if (g.out_class) g.out_class[row] = best + 1;
    if (g.out_prob) g.out_prob[row] = total == 0.f ? 0.f : 1.f / total;
}

// the label of a row: -1 without a class (0), or with a number that is no class (counted)
__device__ __forceinline__ int softmax_label(const Softmax &g, uint64_t row, bool &bad)
{
    if (!g.labels) return -1;
    const int l = g.labels[row];
    bad = l < 0 || l > g.cols;
    return bad ? -1 : l - 1;
}

// Bound by memory: 250 000 x 1564 float32 scores with a bfloat16 gradient 424 us, 5.5 TB/s.
template <class T, int TPR, int NQ, bool NT> __global__ __launch_bounds__(BLOCK) void softmax_kernel(const Softmax g)
{
    __shared__ float red[2 * BLOCK / WAVE];
    Team<TPR> team{red};
    constexpr int RPB = BLOCK / TPR;
    const int t = threadIdx.x % TPR;
    const uint64_t row = g.first + (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row >= g.n) return;
    const T *s = (const T *)g.s + row * g.lds;
    f32x4 x[NQ];
    load_row<T, TPR, NQ>(s, t, g.cols, -INFINITY, x);
    bool bad = false;
    const int label = softmax_label(g, row, bad);
    const float at = label >= 0 && g.loss ? (float)s[label] : 0.f;  // here, before anybody writes: grad may be s
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NQ; i++) top = fmaxf(top, fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])));
    top = team.max(top);
    int best = 0;
    if (g.out_class) {
        int first = 0x7fffffff;                                    // the lowest class of the maximum
#pragma unroll
        for (int i = NQ - 1; i >= 0; i--)
#pragma unroll
            for (int e = 3; e >= 0; e--)
                if (x[i][e] == top) first = quad_col<TPR, NQ>(i, t) + e;
        const float low = -team.max(first == 0x7fffffff ? -INFINITY : -(float)first);   // cols <= 2^20: exact in a float
        best = top > -INFINITY && low < (float)g.cols ? (int)low : 0;      // -inf is ruled out, behind a NaN too: class 1 then
    }
    const float shift = top == -INFINITY ? 0.f : top;
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[i][e] = expf(x[i][e] - shift);
            z += x[i][e];
        }
    z = team.sum(z);
    if (t == 0) softmax_row(g, row, shift, z, best, label, bad, at);
    if (g.grad) {
        const float f = label < 0 || z == 0.f ? 0.f : g.scale / z;
        const bool none = label < 0 || z == 0.f;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int col = quad_col<TPR, NQ>(i, t);
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = none ? 0.f : col + e == label ? x[i][e] * f - g.scale : x[i][e] * f;
            store4_typed<NT>(g.grad, g.grad_type, row * g.ldg + col, quad_left<TPR, NQ>(i, col, g.cols), d);
        }
    }
}

template <class T> __global__ __launch_bounds__(LONG) void softmax_long_kernel(const Softmax g)
{
    __shared__ float red[2 * LONG / WAVE];
    Team<LONG> team{red};
    for (uint64_t row = blockIdx.x; row < g.n; row += gridDim.x) {
        const T *s = (const T *)g.s + row * g.lds;
        bool bad = false;
        const int label = softmax_label(g, row, bad);
        float top = -INFINITY;
        for (int c = threadIdx.x; c < g.cols; c += LONG) top = fmaxf(top, (float)s[c]);
        top = team.max(top);
        const float shift = top == -INFINITY ? 0.f : top;
        float z = 0.f, first = INFINITY;
        for (int c = threadIdx.x; c < g.cols; c += LONG) {
            const float v = (float)s[c];
            if (v == top && first == INFINITY) first = (float)c;
            z += expf(v - shift);
        }
        z = team.sum(z);
        const float low = -team.max(-first);
        const float at = label >= 0 ? (float)s[label] : 0.f;
        if (g.grad) {
            __syncthreads();                                           // grad may be s: everybody has read the label's score
            const bool none = label < 0 || z == 0.f;
            const float f = none ? 0.f : g.scale / z;
            for (int c = threadIdx.x; c < g.cols; c += LONG) {
                const float p = none ? 0.f : expf((float)s[c] - shift) * f;
                store4_typed(g.grad, g.grad_type, row * g.ldg + c, 1, f32x4{!none && c == label ? p - g.scale : p, 0.f, 0.f, 0.f});
            }
        }
        if (threadIdx.x == 0) softmax_row(g, row, shift, z, top > -INFINITY && low < (float)g.cols ? (int)low : 0, label, bad, at);
    }
}

// ------------------------------------------------------------------------------------------------ launches
constexpr int BLOCK_COLS = 8192;

// LAUNCH(TPR, NQ): the narrowest team whose rows fit, and its quads a thread
#define OPAL_TEAMS(LAUNCH, cols)                                  \
    if ((cols) <= 64) { LAUNCH(16, 1); }                          \
    else if ((cols) <= 128) { LAUNCH(16, 2); }                    \
    else if ((cols) <= 256) { LAUNCH(32, 2); }                    \
    else if ((cols) <= 384) { LAUNCH(32, 3); }                    \
    else if ((cols) <= 512) { LAUNCH(32, 4); }                    \
    else if ((cols) <= 768) { LAUNCH(64, 3); }                    \
    else if ((cols) <= 1024) { LAUNCH(64, 4); }                   \
    else if ((cols) <= 1280) { LAUNCH(64, 5); }                   \
    else if ((cols) <= 1536) { LAUNCH(64, 6); }                   \
    else if ((cols) <= 1792) { LAUNCH(64, 7); }                   \
    else if ((cols) <= 2048) { LAUNCH(64, 8); }                   \
    else if ((cols) <= 4096) { LAUNCH(256, 4); }                  \
    else if ((cols) <= 6144) { LAUNCH(256, 6); }                  \
    else { LAUNCH(256, 8); }

static unsigned row_grid(uint64_t n, int rows_per_block, int cus, int blocks_per_cu)
{
    return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>((n + rows_per_block - 1) / rows_per_block, (uint64_t)cus * blocks_per_cu));
}

// A launch has less than 2^32 threads: rows beyond 2^23 blocks are another launch's.  One row a team: fewer blocks that go through
// the rows took 454 .. 526 us where this takes 423 (250 000 x 1564).
template <class G, class Launch> static void launch_rows(G g, int rows_per_block, Launch &&launch)
{
    const uint64_t most = (uint64_t)rows_per_block << 23;
    for (g.first = 0; g.first < g.n; g.first += most)
        launch(g, dim3((unsigned)((std::min(g.n - g.first, most) + rows_per_block - 1) / rows_per_block)));
}

// Results of more than the 256 MiB that the memory-side cache holds are written past it: 250 000 rows of 1564 in bf16, 423 -> 408 us.
static bool stream_out(uint64_t n, uint64_t cols, int type) { return n * cols * type_bytes(type) > (256u << 20); }

template <class T> static void run_norm(const Norm &g, int cus, hipStream_t st)
{
#define L(TPR, NQ)                                                                                               \
    launch_rows(g, BLOCK / TPR, [&](const Norm &q, dim3 blocks) {                                                  \
        if (nt) hipLaunchKernelGGL((norm_kernel<T, TPR, NQ, true>), blocks, dim3(BLOCK), 0, st, q);                \
        else hipLaunchKernelGGL((norm_kernel<T, TPR, NQ, false>), blocks, dim3(BLOCK), 0, st, q);                  \
    })
    const bool nt = stream_out(g.n, g.cols, g.y_type);
    if (g.cols <= BLOCK_COLS) { OPAL_TEAMS(L, g.cols) }
    else hipLaunchKernelGGL(norm_long_kernel<T>, dim3(row_grid(g.n, 1, cus, 2)), dim3(LONG), 0, st, g);
#undef L
}

template <class T> static void run_softmax(const Softmax &g, int cus, hipStream_t st)
{
#define L(TPR, NQ)                                                                                               \
    launch_rows(g, BLOCK / TPR, [&](const Softmax &q, dim3 blocks) {                                                  \
        if (nt) hipLaunchKernelGGL((softmax_kernel<T, TPR, NQ, true>), blocks, dim3(BLOCK), 0, st, q);                \
        else hipLaunchKernelGGL((softmax_kernel<T, TPR, NQ, false>), blocks, dim3(BLOCK), 0, st, q);                  \
    })
    const bool nt = g.grad && stream_out(g.n, g.cols, g.grad_type);
    if (g.cols <= BLOCK_COLS) { OPAL_TEAMS(L, g.cols) }
    else hipLaunchKernelGGL(softmax_long_kernel<T>, dim3(row_grid(g.n, 1, cus, 2)), dim3(LONG), 0, st, g);
#undef L
}

// Blocks of the backward pass, which is the number of partial sums.  Many rows: enough waves to fill the card (two blocks a CU), four rows a
// team at least, below which the partial sums would be as much to read as the rows.  Few: a row a team, since rows in turn are 2 us each: 500 x 356
// 10.4 us a call against 15.8 with four, 5000 x 356 12.0 against 17.5.  Up to two rows a team: one block (64 x 356 9.6 against 10.2).
constexpr uint64_t NORM_BACK_BLOCKS = 512;
static uint64_t norm_back_blocks(uint64_t n, uint32_t cols)
{
    if (cols > BLOCK_COLS) return std::min<uint64_t>((n + 63) / 64, 64);
#define ROWS(TPR, NQ) rows = back_threads(TPR, NQ) / TPR
    uint64_t rows;
    OPAL_TEAMS(ROWS, cols)
#undef ROWS
    if (n <= 2 * rows) return n > 0;
    return std::max(std::min<uint64_t>((n + rows - 1) / rows, 256), std::min<uint64_t>((n + 4 * rows - 1) / (4 * rows), cols <= 2048 ? NORM_BACK_BLOCKS : 2 * NORM_BACK_BLOCKS));
}
// One block needs no sum behind it, and no workspace.
static bool norm_back_alone(uint64_t n, uint32_t cols) { return cols <= BLOCK_COLS && norm_back_blocks(n, cols) == 1; }

template <class TX, class TY> static void run_norm_back(const NormBack &g, unsigned blocks, int cus, hipStream_t st)
{
#define L(TPR, NQ) hipLaunchKernelGGL((norm_back_kernel<TX, TY, TPR, NQ>), dim3(blocks), dim3(back_threads(TPR, NQ)), 0, st, g)
    if (g.cols <= BLOCK_COLS) { OPAL_TEAMS(L, g.cols) }
    else {
        if (g.part) hipLaunchKernelGGL((norm_cols_kernel<TX, TY>), dim3((g.cols + BLOCK - 1) / BLOCK, blocks), dim3(BLOCK), 0, st, g, (g.n + blocks - 1) / blocks);
        if (g.dx) hipLaunchKernelGGL((norm_back_long_kernel<TX, TY>), dim3(row_grid(g.n, 1, cus, 2)), dim3(LONG), 0, st, g);
    }
#undef L
}

template <class TX> static void run_norm_back_x(const NormBack &g, int dy_type, unsigned blocks, int cus, hipStream_t st)
{
    if (dy_type == OPAL_F32) run_norm_back<TX, float>(g, blocks, cus, st);
    else if (dy_type == OPAL_F16) run_norm_back<TX, f16_t>(g, blocks, cus, st);
    else run_norm_back<TX, bf16_t>(g, blocks, cus, st);
}

// ------------------------------------------------------------------------------------------------ argument checks
static int bad_arg(opal_ctx *ctx, const char *who, const std::string &what) { return opal::fail(ctx, OPAL_EINVAL, std::string(who) + ": " + what); }

constexpr uint64_t MAX_COLS = 1u << 20, MAX_ROWS = 1ull << 31, MAX_LD = 1u << 21;

static int check_matrix(opal_ctx *ctx, const char *who, const char *name, const void *p, int type, uint64_t ld, uint64_t rows, uint64_t cols, bool optional = false)
{
    if (!p) return optional || rows == 0 ? OPAL_OK : bad_arg(ctx, who, std::string("null ") + name);
    if (!type_ok(type)) return bad_arg(ctx, who, std::string("unknown element type of ") + name);
    if (ld < cols || ld > MAX_LD) return bad_arg(ctx, who, std::string("the row stride of ") + name + " must lie between its columns and 2^21");
    if (reinterpret_cast<uintptr_t>(p) % type_bytes(type)) return bad_arg(ctx, who, std::string(name) + " is not aligned to its element type");
    return OPAL_OK;
}

// an output over an input: the same rows, each element written by the thread that has read it
static int check_in_place(opal_ctx *ctx, const char *who, const char *names, const void *out, int out_type, uint64_t ld_out, const void *in, int in_type, uint64_t ld_in)
{
    if (!out || out != in || (out_type == in_type && ld_out == ld_in)) return OPAL_OK;
    return bad_arg(ctx, who, std::string(names) + " in the same place need the same type and row stride");
}

static int check_shape(opal_ctx *ctx, const char *who, uint64_t n, uint64_t cols, const char *what)
{
    if (cols < 1 || cols > MAX_COLS) return bad_arg(ctx, who, std::string("need 1 <= ") + what + " <= 2^20");
    if (n >= MAX_ROWS) return bad_arg(ctx, who, "need n < 2^31 rows");
    return OPAL_OK;
}

}  // namespace opal_head

using namespace opal_head;

#define OPAL_TRY(call)          \
    do {                        \
        const int rc__ = (call); \
        if (rc__) return rc__;  \
    } while (0)

extern "C" int opal_layer_norm(opal_ctx *ctx, const void *d_x, int x_type, uint64_t ldx, const float *d_gamma, const float *d_beta,
                               uint64_t n, uint32_t cols, float eps, void *d_y, int y_type, uint64_t ldy, float *d_mean, float *d_rstd)
{
    static const char *who = "opal_layer_norm";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, cols, "cols"));
    if (!(eps > 0.f) || !std::isfinite(eps)) return bad_arg(ctx, who, "eps must be positive and finite");
    OPAL_TRY(check_matrix(ctx, who, "x", d_x, x_type, ldx, n, cols));
    OPAL_TRY(check_matrix(ctx, who, "y", d_y, y_type, ldy, n, cols));
    OPAL_TRY(check_in_place(ctx, who, "x and y", d_y, y_type, ldy, d_x, x_type, ldx));
    if (n == 0) return OPAL_OK;
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const Norm g{d_x, ldx, d_gamma, d_beta, n, (int)cols, eps, d_y, y_type, ldy, d_mean, d_rstd, 0};
    if (x_type == OPAL_F32) run_norm<float>(g, ctx->num_cus, ctx->stream);
    else if (x_type == OPAL_F16) run_norm<f16_t>(g, ctx->num_cus, ctx->stream);
    else run_norm<bf16_t>(g, ctx->num_cus, ctx->stream);
    OPAL_HIP_CHECK(ctx, hipGetLastError());
    return OPAL_OK;
}

extern "C" uint64_t opal_layer_norm_backward_workspace(uint64_t n, uint32_t cols)
{
    if (n >= MAX_ROWS || cols < 1 || cols > MAX_COLS) return 0;      // what the call refuses
    return norm_back_alone(n, cols) ? 0 : norm_back_blocks(n, cols) * 2 * cols * sizeof(float);
}

extern "C" int opal_layer_norm_backward(opal_ctx *ctx, const void *d_dy, int dy_type, uint64_t lddy, const void *d_x, int x_type, uint64_t ldx,
                                        const float *d_gamma, const float *d_mean, const float *d_rstd, uint64_t n, uint32_t cols, void *d_dx,
                                        int dx_type, uint64_t lddx, float *d_dgamma, float *d_dbeta, void *d_work, uint64_t work_bytes)
{
    static const char *who = "opal_layer_norm_backward";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, cols, "cols"));
    OPAL_TRY(check_matrix(ctx, who, "dy", d_dy, dy_type, lddy, n, cols));
    OPAL_TRY(check_matrix(ctx, who, "x", d_x, x_type, ldx, n, cols));
    OPAL_TRY(check_matrix(ctx, who, "dx", d_dx, dx_type, lddx, n, cols, true));
    OPAL_TRY(check_in_place(ctx, who, "x and dx", d_dx, dx_type, lddx, d_x, x_type, ldx));
    OPAL_TRY(check_in_place(ctx, who, "dy and dx", d_dx, dx_type, lddx, d_dy, dy_type, lddy));
    if (n && (!d_mean || !d_rstd)) return bad_arg(ctx, who, "null mean or rstd");
    const bool sums = d_dgamma || d_dbeta, alone = norm_back_alone(n, cols);
    const uint64_t blocks = norm_back_blocks(n, cols), need = opal_layer_norm_backward_workspace(n, cols);
    if (sums && need && (!d_work || work_bytes < need))
        return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": the workspace is smaller than opal_layer_norm_backward_workspace says");
    if (reinterpret_cast<uintptr_t>(d_work) % 16) return bad_arg(ctx, who, "the workspace must be 16-byte aligned");
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    float *part = sums && !alone ? (float *)d_work : nullptr;
    if (n && (sums || d_dx)) {
        const NormBack g{d_dy, lddy, d_x, ldx, d_gamma, d_mean, d_rstd, n, (int)cols, d_dx, dx_type, lddx, part, alone ? d_dgamma : nullptr, alone ? d_dbeta : nullptr, d_dx && stream_out(n, cols, dx_type)};
        if (x_type == OPAL_F32) run_norm_back_x<float>(g, dy_type, (unsigned)blocks, ctx->num_cus, ctx->stream);
        else if (x_type == OPAL_F16) run_norm_back_x<f16_t>(g, dy_type, (unsigned)blocks, ctx->num_cus, ctx->stream);
        else run_norm_back_x<bf16_t>(g, dy_type, (unsigned)blocks, ctx->num_cus, ctx->stream);
        OPAL_HIP_CHECK(ctx, hipGetLastError());
    }
    if (sums && !alone) {
        hipLaunchKernelGGL(sum_parts_kernel, dim3((2 * cols + 15) / 16), dim3(1024), 0, ctx->stream, part, (uint32_t)blocks, cols, d_dgamma, d_dbeta);
        OPAL_HIP_CHECK(ctx, hipGetLastError());
    }
    return OPAL_OK;
}

static int softmax(opal_ctx *ctx, const char *who, const void *d_scores, int type, uint64_t ld, uint64_t n, uint32_t K, const int32_t *d_labels, float scale,
                   float *d_loss, void *d_grad, int grad_type, uint64_t ldg, int32_t *d_class, float *d_prob)
{
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, K, "K"));
    OPAL_TRY(check_matrix(ctx, who, "scores", d_scores, type, ld, n, K));
    OPAL_TRY(check_matrix(ctx, who, "grad", d_grad, grad_type, ldg, n, K, true));
    OPAL_TRY(check_in_place(ctx, who, "scores and grad", d_grad, grad_type, ldg, d_scores, type, ld));
    if (n == 0) return OPAL_OK;
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const Softmax g{d_scores, ld, n, (int)K, d_labels, scale, d_loss, d_grad, grad_type, ldg, d_class, d_prob, ctx->d_queue + Q_BAD_LABEL, 0};
    if (type == OPAL_F32) run_softmax<float>(g, ctx->num_cus, ctx->stream);
    else if (type == OPAL_F16) run_softmax<f16_t>(g, ctx->num_cus, ctx->stream);
    else run_softmax<bf16_t>(g, ctx->num_cus, ctx->stream);
    OPAL_HIP_CHECK(ctx, hipGetLastError());
    return OPAL_OK;
}

extern "C" int opal_softmax_loss(opal_ctx *ctx, const void *d_scores, int type, uint64_t ld, uint64_t n, uint32_t K, const int32_t *d_labels,
                                 float scale, float *d_loss, void *d_grad, int grad_type, uint64_t ldg)
{
    static const char *who = "opal_softmax_loss";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    if (n && !d_labels) return bad_arg(ctx, who, "null labels");
    if (n && !d_loss && !d_grad) return bad_arg(ctx, who, "neither the loss nor the gradient is asked for");
    return softmax(ctx, who, d_scores, type, ld, n, K, d_labels, scale, d_loss, d_grad, grad_type, ldg, nullptr, nullptr);
}

extern "C" int opal_softmax_class(opal_ctx *ctx, const void *d_scores, int type, uint64_t ld, uint64_t n, uint32_t K, int32_t *d_out_class, float *d_out_prob)
{
    static const char *who = "opal_softmax_class";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    if (n && !d_out_class) return bad_arg(ctx, who, "null d_out_class");
    return softmax(ctx, who, d_scores, type, ld, n, K, nullptr, 0.f, nullptr, nullptr, OPAL_F32, 0, d_out_class, d_out_prob);
}

// ------------------------------------------------------------------------------------------------ matrix products
static hipError_t launch(const Linear &g, int type, int product, int tile, bool dma, hipStream_t st)
{
    if (type == OPAL_F32) return launch_linear<float>(g, product, tile, dma, st);
    if (type == OPAL_F16) return launch_linear<f16_t>(g, product, tile, dma, st);
    return launch_linear<bf16_t>(g, product, tile, dma, st);
}

static void set_tiles(Linear &g, int tile)
{
    g.tm = (uint32_t)((g.M + TILE_M[tile] - 1) / TILE_M[tile]);
    g.tn = (uint32_t)((g.N + TILE_N[tile] - 1) / TILE_N[tile]);
}

// 16-byte chunks straight into LDS need matrices and rows that begin on 16 bytes
static bool aligned16(const void *p, uint64_t ld, int type) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * type_bytes(type) % 16 == 0; }

static const char *past(const void *p, uint64_t rows, uint64_t ld, int type) { return p ? (const char *)p + rows * ld * type_bytes(type) : nullptr; }

// the product without its first `rows` rows
static Linear behind(const Linear &g, uint64_t rows, int type)
{
    Linear q = g;
    q.M = g.M - rows;
    q.a = past(g.a, rows, g.lda, type);
    q.res = past(g.res, rows, g.ldr, g.res_type);
    q.y = (void *)past(g.y, rows, g.ldy, g.y_type);
    q.pre_in = past(g.pre_in, rows, g.ldp, type);
    q.pre_out = (void *)past(g.pre_out, rows, g.ldp, type);
    return q;
}

constexpr uint64_t MOST_TILES = 1u << 24;      // of 256 threads in a launch, which has less than 2^32

static int run_rows(opal_ctx *ctx, const Linear &product_of, int type, int product)
{
    Linear g = product_of;
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    // as many rows at a time as the smallest tiles have room for in a launch
    const uint64_t slice = (MOST_TILES - 1) / ((g.N + TILE_N[0] - 1) / TILE_N[0]) * TILE_M[0] / 256 * 256;
    if (g.M > slice) {
        Linear q = g;
        q.M = slice;
        OPAL_TRY(run_rows(ctx, q, type, product));
        return run_rows(ctx, behind(g, slice, type), type, product);
    }
    const bool dma = aligned16(g.a, g.lda, type) && aligned16(g.b, g.ldb, type);
    const int cus = ctx->num_cus;
    // (the two kernels for large products write 32 bits or the operands' type, and read such a residual)
    const bool large = dma && type != OPAL_F32 && (g.y_type == OPAL_F32 || g.y_type == type) && (!g.res || g.res_type == OPAL_F32 || g.res_type == type);
    int tile = product_tile(product, type, g.M, g.N, g.K, cus, large, true);
    g.splits = 1;
    g.ksplit = g.K;
    auto run = [&](Linear &q, int t) {
        if (t == 3) {
            q.few = q.M <= 16 ? 1 : q.M <= 32 ? 2 : 4;
            q.tm = (uint32_t)((q.M + 16 * q.few - 1) / (16 * q.few));
            q.tn = (uint32_t)((q.N + 15) / 16);
        } else set_tiles(q, t);
        q.items = q.tm * q.tn;
        q.blocks = std::min<uint32_t>(q.items, cus);
        return launch(q, type, product, t, dma, ctx->stream);
    };
    // 256 x 256 tiles come in rounds of one a CU.  A last round of up to a quarter of the CUs goes to smaller tiles instead, in a
    // launch of its own: 100 000 x 512 x 1564 (3.05 rounds) 239 -> 220 us; with two fifths, 60 001 x 1563 x 512 (6.43), 245 -> 256.
    const uint64_t tn = (g.N + TILE_M[2] - 1) / TILE_M[2], tiles = tiles_of(g.M, g.N, 2), rounds = tiles / cus;
    const uint64_t rows = rounds * cus / tn * TILE_M[2];
    if (tile == 2 && rounds && rows < g.M && (tiles - rows / TILE_M[2] * tn) * 4 <= (uint64_t)cus) {
        Linear q = g;
        q.M = rows;
        OPAL_HIP_CHECK(ctx, run(q, 2));
        g = behind(g, rows, type);
        tile = product_tile(product, type, g.M, g.N, g.K, cus, large, false);
    }
    OPAL_HIP_CHECK(ctx, run(g, tile));
    return OPAL_OK;
}

extern "C" int opal_linear(opal_ctx *ctx, const void *d_x, uint64_t ldx, const void *d_w, uint64_t ldw, int type, const float *d_bias,
                           int activation, const void *d_res, int res_type, uint64_t ldr, uint64_t n, uint32_t in, uint32_t out,
                           void *d_y, int y_type, uint64_t ldy, void *d_pre, uint64_t ldp)
{
    static const char *who = "opal_linear";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, in, "in"));
    OPAL_TRY(check_shape(ctx, who, n, out, "out"));
    if (activation < ACT_NONE || activation > ACT_GELU) return bad_arg(ctx, who, "unknown activation");
    OPAL_TRY(check_matrix(ctx, who, "x", d_x, type, ldx, n, in));
    OPAL_TRY(check_matrix(ctx, who, "w", d_w, type, ldw, out, in));
    OPAL_TRY(check_matrix(ctx, who, "the residual", d_res, res_type, ldr, n, out, true));
    OPAL_TRY(check_matrix(ctx, who, "y", d_y, y_type, ldy, n, out));
    OPAL_TRY(check_matrix(ctx, who, "pre", d_pre, type, ldp, n, out, true));
    if (n == 0) return OPAL_OK;
    OPAL_TRY(check_in_place(ctx, who, "the residual and y", d_y, y_type, ldy, d_res, res_type, ldr));
    if (d_y == d_x || d_y == d_w || d_y == d_pre || (d_pre && (d_pre == d_x || d_pre == d_w || d_pre == d_res))) return bad_arg(ctx, who, "y and pre need places of their own");
    Linear g{};
    g.a = (const char *)d_x; g.lda = ldx; g.b = (const char *)d_w; g.ldb = ldw;
    g.M = n; g.N = out; g.K = in;
    g.bias = d_bias; g.act = activation;
    g.res = d_res; g.res_type = res_type; g.ldr = ldr;
    g.y = d_y; g.y_type = y_type; g.ldy = ldy;
    g.pre_out = d_pre; g.ldp = ldp;
    return run_rows(ctx, g, type, FWD);
}

extern "C" int opal_linear_grad_input(opal_ctx *ctx, const void *d_dy, uint64_t lddy, const void *d_w, uint64_t ldw, int type, const void *d_pre,
                                      uint64_t ldp, int activation, const void *d_res, int res_type, uint64_t ldr, uint64_t n, uint32_t in,
                                      uint32_t out, void *d_dx, int dx_type, uint64_t lddx)
{
    static const char *who = "opal_linear_grad_input";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, in, "in"));
    OPAL_TRY(check_shape(ctx, who, n, out, "out"));
    if (activation < ACT_NONE || activation > ACT_GELU) return bad_arg(ctx, who, "unknown activation");
    if (activation != ACT_NONE && n && !d_pre) return bad_arg(ctx, who, "an activation's gradient needs its pre-activation");
    OPAL_TRY(check_matrix(ctx, who, "dy", d_dy, type, lddy, n, out));
    OPAL_TRY(check_matrix(ctx, who, "w", d_w, type, ldw, out, in));
    OPAL_TRY(check_matrix(ctx, who, "pre", d_pre, type, ldp, n, in, true));
    OPAL_TRY(check_matrix(ctx, who, "the residual", d_res, res_type, ldr, n, in, true));
    OPAL_TRY(check_matrix(ctx, who, "dx", d_dx, dx_type, lddx, n, in));
    if (n == 0) return OPAL_OK;
    OPAL_TRY(check_in_place(ctx, who, "the residual and dx", d_dx, dx_type, lddx, d_res, res_type, ldr));
    if (d_dx == d_dy || d_dx == d_w || d_dx == d_pre) return bad_arg(ctx, who, "dx needs a place of its own");
    Linear g{};
    g.a = (const char *)d_dy; g.lda = lddy; g.b = (const char *)d_w; g.ldb = ldw;
    g.M = n; g.N = in; g.K = out;
    g.act = activation; g.pre_in = d_pre; g.ldp = ldp;
    g.res = d_res; g.res_type = res_type; g.ldr = ldr;
    g.y = d_dx; g.y_type = dx_type; g.ldy = lddx;
    return run_rows(ctx, g, type, GIN);
}

extern "C" uint64_t opal_linear_grad_weight_workspace(uint64_t n, uint32_t in, uint32_t out, int type)
{
    if (!type_ok(type) || n >= MAX_ROWS || in < 1 || out < 1 || in > MAX_COLS || out > MAX_COLS) return 0;      // what the call refuses
    const Splits s = weight_splits(n, in, out, type);
    return s.splits > 1 ? s.splits * ((uint64_t)in * out + out) * sizeof(float) : 0;
}

namespace opal_head {
// The sum of the splits' matrices and of their row sums: [splits][each] -> dw (rows of `cols`), [splits][out] -> db (or null).  Reads what the
// product has just written.  A thread adds up four neighbouring values of every G-th split, eight loads under way; G threads, which
// small matrices need to fill the card, then add up in LDS: always in the same order.
template <int G> __global__ __launch_bounds__(BLOCK) void sum_splits_kernel(const float *part, const float *rows, uint32_t splits, uint64_t each, uint32_t cols,
                                                                            uint32_t out, float *dw, uint64_t ld, float *db)
{
    constexpr int QUADS = BLOCK / G;
    __shared__ f32x4 red[G][QUADS];
    const int q = threadIdx.x % QUADS, group = threadIdx.x / QUADS;
    const uint64_t quads = (each + 3) / 4, i = (uint64_t)blockIdx.x * QUADS + q, r = i - quads;
    const bool row = i >= quads;               // of the row sums, one a thread
    const int left = !row ? (int)std::min<uint64_t>(each - i * 4, 4) : db && r < out ? 1 : 0;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (left == 4) {
#pragma unroll 8
        for (uint32_t p = group; p < splits; p += G) s += load4(part + p * each + i * 4);
    } else if (left) {
        const float *from = row ? rows + r : part + i * 4;
        const uint64_t stride = row ? out : each;
#pragma unroll 8
        for (uint32_t p = group; p < splits; p += G) s += load4_typed(from, OPAL_F32, p * stride, left);
    }
    red[group][q] = s;
    __syncthreads();
    if (group || !left) return;
#pragma unroll 8
    for (int p = 1; p < G; p++) s += red[p][q];
    if (row) db[r] = s[0];
    else if (ld == cols) store4_typed(dw, OPAL_F32, i * 4, left, s);
    else
        for (int e = 0; e < left; e++) {
            const uint64_t at = i * 4 + e;
            dw[at / cols * ld + at % cols] = s[e];
        }
}
}  // namespace opal_head

extern "C" int opal_linear_grad_weight(opal_ctx *ctx, const void *d_dy, uint64_t lddy, const void *d_x, uint64_t ldx, int type, uint64_t n, uint32_t in,
                                       uint32_t out, float *d_dw, uint64_t lddw, float *d_dbias, void *d_work, uint64_t work_bytes)
{
    static const char *who = "opal_linear_grad_weight";
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, in, "in"));
    OPAL_TRY(check_shape(ctx, who, n, out, "out"));
    OPAL_TRY(check_matrix(ctx, who, "dy", d_dy, type, lddy, n, out));
    OPAL_TRY(check_matrix(ctx, who, "x", d_x, type, ldx, n, in));
    OPAL_TRY(check_matrix(ctx, who, "dw", d_dw, OPAL_F32, lddw, out, in));
    if (!type_ok(type)) return bad_arg(ctx, who, "unknown element type");
    const uint64_t need = opal_linear_grad_weight_workspace(n, in, out, type);
    if (need && (!d_work || work_bytes < need)) return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": the workspace is smaller than opal_linear_grad_weight_workspace says");
    if (reinterpret_cast<uintptr_t>(d_work) % 16) return bad_arg(ctx, who, "the workspace must be 16-byte aligned");
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const Splits s = weight_splits(n, in, out, type);
    const uint64_t each = (uint64_t)in * out;
    float *part = s.splits > 1 ? (float *)d_work : nullptr, *rows = part ? part + s.splits * each : nullptr;
    const bool dma = aligned16(d_dy, lddy, type) && aligned16(d_x, ldx, type);
    const int tile = s.tile == 2 && !dma ? 1 : s.tile;
    Linear g{};
    g.a = (const char *)d_dy; g.lda = lddy; g.b = (const char *)d_x; g.ldb = ldx;
    g.M = out; g.N = in; g.K = n;
    if (tiles_of(g.M, g.N, tile) * s.splits >= MOST_TILES) return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": in times out is too large for one call");
    set_tiles(g, tile);
    g.splits = (uint32_t)s.splits;
    g.ksplit = s.rows;
    g.items = g.tm * g.tn * g.splits;
    g.blocks = std::min<uint32_t>(g.items, ctx->num_cus);
    g.y = part ? part : d_dw; g.y_type = OPAL_F32; g.ldy = part ? in : lddw; g.y_split = each;
    g.colsum = d_dbias ? (part ? rows : d_dbias) : nullptr;
    OPAL_HIP_CHECK(ctx, launch(g, type, GWT, tile, dma, ctx->stream));
    if (part) {
        // 300 000 x 63 x 64 (512 splits of 4032 values) 138 -> 22 us with 64 threads for each four, 20 000 x 355 x 128 (42 of 45 440) 24 -> 14 with 16
        const uint64_t work = (each + 3) / 4 + out;
#define L(G)                                                                                                                              \
    hipLaunchKernelGGL(sum_splits_kernel<G>, dim3((unsigned)((work + BLOCK / G - 1) / (BLOCK / G))), dim3(BLOCK), 0, ctx->stream, part, rows, \
                       (uint32_t)s.splits, each, in, out, d_dw, lddw, d_dbias)
        if (work <= 2048) L(64);
        else if (work <= 16384) L(16);
        else L(4);
#undef L
        OPAL_HIP_CHECK(ctx, hipGetLastError());
    }
    return OPAL_OK;
}
