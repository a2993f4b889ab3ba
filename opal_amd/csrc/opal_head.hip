// Row operators of the score head: layer norm (forward, backward with the reduction of the weight's gradient) and the softmax loss
// over the class scores; and the C entry points of these and of the matrix products (opal_linear.h).
//
//   layer norm   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), y = (x - m) r g + b
//   backward     h = dy g, xh = (x - m) r:  dx = r (h - mean(h) - xh mean(h xh));  dg = sum_rows dy xh,  db = sum_rows dy
//   softmax      e_j = exp(s_j - max), Z = sum e_j:  loss = log Z + max - s_label, grad_j = scale (e_j / Z - [j is the label])
//
// A row of up to 2048 columns belongs to a wave, which holds it in registers (one read of memory, sums over the wave's lanes);
// up to 8192 to a block of 256 threads in the same way; a longer one is read again by a block of 1024 for each pass.
#include <algorithm>
#include <cmath>
#include <string>

#include "opal_linear.h"

namespace opal_head {

constexpr int BLOCK = 256;

// Sums and maxima over the TPR threads of a row: a wave, or the whole block (red: one float per wave and value, two buffers in
// turn so that a block needs one barrier per reduction).
template <int TPR> struct Team {
    float *red;
    int turn = 0;
    __device__ __forceinline__ float join(float v, bool take_max)
    {
        v = take_max ? wave_max(v) : wave_sum(v);
        if constexpr (TPR == WAVE) return v;
        else {
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

// A thread's share of a row: quads i * TPR + t, i < NQ = ceil(cols / (4 TPR)); all but the last are whole.
template <int TPR, int NQ> __device__ __forceinline__ int quad_col(int i, int t) { return (i * TPR + t) * 4; }
template <int NQ> __device__ __forceinline__ int quad_left(int i, int col, int cols)
{
    return i < NQ - 1 ? 4 : cols - col;
}

template <class T> constexpr int type_of() { return __is_same(T, float) ? OPAL_F32 : __is_same(T, f16_t) ? OPAL_F16 : OPAL_BF16; }

template <class T, int TPR, int NQ>
__device__ __forceinline__ void load_row(const T *row, int t, int cols, float fill, f32x4 (&v)[NQ])
{
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int col = quad_col<TPR, NQ>(i, t);
        v[i] = load4_typed(row, type_of<T>(), col, quad_left<NQ>(i, col, cols), fill);
    }
}

struct Norm {
    const void *x; uint64_t ldx;
    const float *gamma, *beta;
    uint64_t n; int cols; float eps;
    void *y; int y_type; uint64_t ldy;
    float *mean, *rstd;
};

__device__ __forceinline__ f32x4 param4(const float *p, int col, int left, float none)
{
    return p ? load4_typed(p, OPAL_F32, col, left, none) : f32x4{none, none, none, none};
}

template <class T, int TPR, int NQ> __global__ __launch_bounds__(BLOCK) void norm_kernel(const Norm g)
{
    __shared__ float red[2 * BLOCK / WAVE];
    Team<TPR> team{red};
    constexpr int RPB = BLOCK / TPR;
    const int t = threadIdx.x % TPR;
    const float cols = (float)g.cols;
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < g.n; row += (uint64_t)gridDim.x * RPB) {
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
                if (quad_left<NQ>(i, quad_col<TPR, NQ>(i, t), g.cols) > e) s += x[i][e] * x[i][e];
            }
        const float rstd = 1.f / sqrtf(team.sum(s) / cols + g.eps);
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int col = quad_col<TPR, NQ>(i, t), left = quad_left<NQ>(i, col, g.cols);
            const f32x4 ga = param4(g.gamma, col, left, 1.f), be = param4(g.beta, col, left, 0.f);
            f32x4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = x[i][e] * rstd * ga[e] + be[e];
            store4_typed(g.y, g.y_type, row * g.ldy + col, left, y);
        }
        if (t == 0) {
            if (g.mean) g.mean[row] = mean;
            if (g.rstd) g.rstd[row] = rstd;
        }
    }
}

constexpr int LONG = 1024;                // threads on a row that does not fit the registers

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
    float *part;                               // [blocks][2][cols]: dgamma, dbeta; null: not wanted
};

// Every thread keeps the sums of its own columns over the rows that its team visits; the teams of a block add theirs up in
// order, and norm_sums_kernel adds the blocks': no atomics, the same bits every time.
template <class TX, class TY, int TPR, int NQ> __global__ __launch_bounds__(BLOCK) void norm_back_kernel(const NormBack g)
{
    __shared__ float red[2 * BLOCK / WAVE];
    __shared__ f32x4 both[TPR == BLOCK ? 1 : 2 * NQ * TPR];
    Team<TPR> team{red};
    constexpr int RPB = BLOCK / TPR;
    const int t = threadIdx.x % TPR;
    const float cols = (float)g.cols;
    f32x4 dg[NQ], db[NQ];
#pragma unroll
    for (int i = 0; i < NQ; i++) dg[i] = db[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < g.n; row += (uint64_t)gridDim.x * RPB) {
        f32x4 x[NQ], h[NQ];
        load_row<TX, TPR, NQ>((const TX *)g.x + row * g.ldx, t, g.cols, 0.f, x);
        load_row<TY, TPR, NQ>((const TY *)g.dy + row * g.lddy, t, g.cols, 0.f, h);
        const float mean = g.mean[row], rstd = g.rstd[row];
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int col = quad_col<TPR, NQ>(i, t), left = quad_left<NQ>(i, col, g.cols);
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
            const int col = quad_col<TPR, NQ>(i, t), left = quad_left<NQ>(i, col, g.cols);
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = rstd * (h[i][e] - s0 - x[i][e] * s1);
            store4_typed(g.dx, g.dx_type, row * g.lddx + col, left, d);
        }
    }
    if (!g.part) return;
    if constexpr (TPR == WAVE) {
        for (int w = 0; w < RPB; w++) {
            if ((int)(threadIdx.x / TPR) == w) {
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
        if ((int)(threadIdx.x / TPR) != RPB - 1) return;      // the last team holds the block's sums
    }
    float *out = g.part + (uint64_t)blockIdx.x * 2 * g.cols;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int col = quad_col<TPR, NQ>(i, t), left = quad_left<NQ>(i, col, g.cols);
        store4_typed(out, OPAL_F32, col, left, dg[i]);
        store4_typed(out, OPAL_F32, (uint64_t)g.cols + col, left, db[i]);
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

// out[c] = sum over parts of part[p * stride + c], c < width, in a fixed order; parts == 0 writes zeros.
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float *part, uint64_t parts, uint64_t stride, uint64_t width, float *out)
{
    __shared__ float acc[16][64];
    const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t col = (uint64_t)blockIdx.x * 64 + c;
    float s = 0.f;
    if (col < width)
        for (uint64_t p = w; p < parts; p += 16) s += part[p * stride + col];
    acc[w][c] = s;
    __syncthreads();
    if (w == 0 && col < width) {
        for (int i = 1; i < 16; i++) s += acc[i][c];
        out[col] = s;
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

template <class T, int TPR, int NQ> __global__ __launch_bounds__(BLOCK) void softmax_kernel(const Softmax g)
{
    __shared__ float red[2 * BLOCK / WAVE];
    Team<TPR> team{red};
    constexpr int RPB = BLOCK / TPR;
    const int t = threadIdx.x % TPR;
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < g.n; row += (uint64_t)gridDim.x * RPB) {
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
            best = low < (float)g.cols ? (int)low : 0;
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
                store4_typed(g.grad, g.grad_type, row * g.ldg + col, quad_left<NQ>(i, col, g.cols), d);
            }
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
        if (threadIdx.x == 0) softmax_row(g, row, shift, z, low < (float)g.cols ? (int)low : 0, label, bad, at);
    }
}

// ------------------------------------------------------------------------------------------------ launches
constexpr int WAVE_COLS = 2048, BLOCK_COLS = 8192;

#define OPAL_NQ_CASES(LAUNCH, TPR, NQ) \
    switch (NQ) {                      \
    case 1: LAUNCH(TPR, 1); break;     \
    case 2: LAUNCH(TPR, 2); break;     \
    case 3: LAUNCH(TPR, 3); break;     \
    case 4: LAUNCH(TPR, 4); break;     \
    case 5: LAUNCH(TPR, 5); break;     \
    case 6: LAUNCH(TPR, 6); break;     \
    case 7: LAUNCH(TPR, 7); break;     \
    default: LAUNCH(TPR, 8); break;    \
    }

static unsigned row_grid(uint64_t n, int rows_per_block, int cus, int blocks_per_cu)
{
    return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>((n + rows_per_block - 1) / rows_per_block, (uint64_t)cus * blocks_per_cu));
}

template <class T> static void run_norm(const Norm &g, int cus, hipStream_t st)
{
#define L(TPR, NQ) hipLaunchKernelGGL((norm_kernel<T, TPR, NQ>), dim3(row_grid(g.n, BLOCK / TPR, cus, 8)), dim3(BLOCK), 0, st, g)
    if (g.cols <= WAVE_COLS) { OPAL_NQ_CASES(L, 64, (g.cols + 255) / 256) }
    else if (g.cols <= BLOCK_COLS) { OPAL_NQ_CASES(L, 256, (g.cols + 1023) / 1024) }
    else hipLaunchKernelGGL(norm_long_kernel<T>, dim3(row_grid(g.n, 1, cus, 2)), dim3(LONG), 0, st, g);
#undef L
}

template <class T> static void run_softmax(const Softmax &g, int cus, hipStream_t st)
{
#define L(TPR, NQ) hipLaunchKernelGGL((softmax_kernel<T, TPR, NQ>), dim3(row_grid(g.n, BLOCK / TPR, cus, 8)), dim3(BLOCK), 0, st, g)
    if (g.cols <= WAVE_COLS) { OPAL_NQ_CASES(L, 64, (g.cols + 255) / 256) }
    else if (g.cols <= BLOCK_COLS) { OPAL_NQ_CASES(L, 256, (g.cols + 1023) / 1024) }
    else hipLaunchKernelGGL(softmax_long_kernel<T>, dim3(row_grid(g.n, 1, cus, 2)), dim3(LONG), 0, st, g);
#undef L
}

// Blocks of the backward pass, which is the number of partial sums: enough to fill the card, and none with less than eight rows
// a team, below which the partial sums would be as much to read as the rows.
constexpr uint64_t NORM_BACK_BLOCKS = 1024;
static uint64_t norm_back_blocks(uint64_t n, uint32_t cols)
{
    if (cols > BLOCK_COLS) return std::min<uint64_t>((n + 63) / 64, 64);
    const uint64_t rpb = cols <= WAVE_COLS ? BLOCK / WAVE : 1;
    return std::min<uint64_t>((n + 8 * rpb - 1) / (8 * rpb), NORM_BACK_BLOCKS);
}

template <class TX, class TY> static void run_norm_back(const NormBack &g, unsigned blocks, int cus, hipStream_t st)
{
#define L(TPR, NQ) hipLaunchKernelGGL((norm_back_kernel<TX, TY, TPR, NQ>), dim3(blocks), dim3(BLOCK), 0, st, g)
    if (g.cols <= WAVE_COLS) { OPAL_NQ_CASES(L, 64, (g.cols + 255) / 256) }
    else if (g.cols <= BLOCK_COLS) { OPAL_NQ_CASES(L, 256, (g.cols + 1023) / 1024) }
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

static void sum_parts(const float *part, uint64_t parts, uint64_t stride, uint64_t width, float *out, hipStream_t st)
{
    hipLaunchKernelGGL(sum_parts_kernel, dim3((unsigned)((width + 63) / 64)), dim3(1024), 0, st, part, parts, stride, width, out);
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
    if (n == 0) return OPAL_OK;
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const Norm g{d_x, ldx, d_gamma, d_beta, n, (int)cols, eps, d_y, y_type, ldy, d_mean, d_rstd};
    if (x_type == OPAL_F32) run_norm<float>(g, ctx->num_cus, ctx->stream);
    else if (x_type == OPAL_F16) run_norm<f16_t>(g, ctx->num_cus, ctx->stream);
    else run_norm<bf16_t>(g, ctx->num_cus, ctx->stream);
    OPAL_HIP_CHECK(ctx, hipGetLastError());
    return OPAL_OK;
}

extern "C" uint64_t opal_layer_norm_backward_workspace(uint64_t n, uint32_t cols)
{
    return norm_back_blocks(n, cols) * 2 * cols * sizeof(float);
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
    if (n && (!d_mean || !d_rstd)) return bad_arg(ctx, who, "null mean or rstd");
    const bool sums = d_dgamma || d_dbeta;
    const uint64_t blocks = norm_back_blocks(n, cols);
    if (sums && n && (!d_work || work_bytes < opal_layer_norm_backward_workspace(n, cols)))
        return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": the workspace is smaller than opal_layer_norm_backward_workspace says");
    if (reinterpret_cast<uintptr_t>(d_work) % 16) return bad_arg(ctx, who, "the workspace must be 16-byte aligned");
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    float *part = sums ? (float *)d_work : nullptr;
    if (n && (sums || d_dx)) {
        const NormBack g{d_dy, lddy, d_x, ldx, d_gamma, d_mean, d_rstd, n, (int)cols, d_dx, dx_type, lddx, part};
        if (x_type == OPAL_F32) run_norm_back_x<float>(g, dy_type, (unsigned)blocks, ctx->num_cus, ctx->stream);
        else if (x_type == OPAL_F16) run_norm_back_x<f16_t>(g, dy_type, (unsigned)blocks, ctx->num_cus, ctx->stream);
        else run_norm_back_x<bf16_t>(g, dy_type, (unsigned)blocks, ctx->num_cus, ctx->stream);
        OPAL_HIP_CHECK(ctx, hipGetLastError());
    }
    if (d_dgamma) sum_parts(part, blocks, 2ull * cols, cols, d_dgamma, ctx->stream);
    if (d_dbeta) sum_parts(part + cols, blocks, 2ull * cols, cols, d_dbeta, ctx->stream);
    OPAL_HIP_CHECK(ctx, hipGetLastError());
    return OPAL_OK;
}

static int softmax(opal_ctx *ctx, const char *who, const void *d_scores, int type, uint64_t ld, uint64_t n, uint32_t K, const int32_t *d_labels, float scale,
                   float *d_loss, void *d_grad, int grad_type, uint64_t ldg, int32_t *d_class, float *d_prob)
{
    if (!ctx) return bad_arg(nullptr, who, "null ctx");
    OPAL_TRY(check_shape(ctx, who, n, K, "K"));
    OPAL_TRY(check_matrix(ctx, who, "scores", d_scores, type, ld, n, K));
    OPAL_TRY(check_matrix(ctx, who, "grad", d_grad, grad_type, ldg, n, K, true));
    if (n == 0) return OPAL_OK;
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const Softmax g{d_scores, ld, n, (int)K, d_labels, scale, d_loss, d_grad, grad_type, ldg, d_class, d_prob, ctx->d_queue + Q_BAD_LABEL};
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

constexpr int TILE[] = {64, 128, 256};

static uint64_t tiles_of(uint64_t M, uint64_t N, int tile) { return ((M + TILE[tile] - 1) / TILE[tile]) * ((N + TILE[tile] - 1) / TILE[tile]); }

// The largest tile that still gives every CU one (256 x 256: half of them, since its kernel is twice as fast): fewer bytes for the
// same sums against idle CUs.
static int pick_tile(uint64_t M, uint64_t N, int cus, bool big)
{
    if (big && tiles_of(M, N, 2) * 2 >= (uint64_t)cus) return 2;
    return tiles_of(M, N, 1) >= (uint64_t)cus ? 1 : 0;
}

static void set_tiles(Linear &g, int tile)
{
    g.tm = (uint32_t)((g.M + TILE[tile] - 1) / TILE[tile]);
    g.tn = (uint32_t)((g.N + TILE[tile] - 1) / TILE[tile]);
}

// 16-byte chunks straight into LDS need matrices and rows that begin on 16 bytes
static bool aligned16(const void *p, uint64_t ld, int type) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * type_bytes(type) % 16 == 0; }

static int run_rows(opal_ctx *ctx, const char *who, Linear &g, int type, int product)
{
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const bool dma = aligned16(g.a, g.lda, type) && aligned16(g.b, g.ldb, type);
    const int tile = pick_tile(g.M, g.N, ctx->num_cus, dma && type != OPAL_F32);
    if (tiles_of(g.M, g.N, tile) >= (1ull << 31)) return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": too many rows times columns for one call");
    set_tiles(g, tile);
    g.splits = 1;
    g.ksplit = g.K;
    g.items = g.tm * g.tn;
    g.blocks = std::min<uint32_t>(g.items, ctx->num_cus);
    OPAL_HIP_CHECK(ctx, launch(g, type, product, tile, dma, ctx->stream));
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
    Linear g{};
    g.a = (const char *)d_x; g.lda = ldx; g.b = (const char *)d_w; g.ldb = ldw;
    g.M = n; g.N = out; g.K = in;
    g.bias = d_bias; g.act = activation;
    g.res = d_res; g.res_type = res_type; g.ldr = ldr;
    g.y = d_y; g.y_type = y_type; g.ldy = ldy;
    g.pre_out = d_pre; g.ldp = ldp;
    return run_rows(ctx, who, g, type, FWD);
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
    Linear g{};
    g.a = (const char *)d_dy; g.lda = lddy; g.b = (const char *)d_w; g.ldb = ldw;
    g.M = n; g.N = in; g.K = out;
    g.act = activation; g.pre_in = d_pre; g.ldp = ldp;
    g.res = d_res; g.res_type = res_type; g.ldr = ldr;
    g.y = d_dx; g.y_type = dx_type; g.ldy = lddx;
    return run_rows(ctx, who, g, type, GIN);
}

// Splits of the sum over the rows, none empty.  256 x 256 tiles: as many as give the 256 CUs a tile each, of at least 16 steps.
// Smaller ones: two blocks per CU, of at least four steps.  The choice does not look at the operands' alignment, so that the workspace
// does not depend on it; unaligned operands take 128 x 128 tiles in the same splits.
struct Splits { int tile; uint64_t splits, rows; };
static Splits weight_splits(uint64_t n, uint32_t in, uint32_t out, int type)
{
    const uint64_t step = STEP_BYTES / type_bytes(type);
    const uint64_t steps = std::max<uint64_t>((n + step - 1) / step, 1);
    const uint64_t big = tiles_of(out, in, 2);
    const bool large = type != OPAL_F32 && in > 128 && out > 128 && steps * big >= 16 * 128;
    const int tile = large ? 2 : in > 64 && out > 64 ? 1 : 0;
    uint64_t s = large ? std::min<uint64_t>(256 / std::min<uint64_t>(big, 256), steps / 16) : std::min<uint64_t>(512 / std::min<uint64_t>(tiles_of(out, in, tile), 512), steps / 4);
    s = std::max<uint64_t>(s, 1);
    const uint64_t per = (steps + s - 1) / s;
    return {tile, (steps + per - 1) / per, per * step};
}

constexpr uint64_t COL_PARTS = 256;       // partial column sums of dy for the bias' gradient
static uint64_t bias_parts(uint64_t n) { return std::min<uint64_t>((n + 31) / 32, COL_PARTS); }

extern "C" uint64_t opal_linear_grad_weight_workspace(uint64_t n, uint32_t in, uint32_t out, int type)
{
    if (!type_ok(type)) return 0;
    const Splits s = weight_splits(n, in, out, type);
    return ((s.splits > 1 ? s.splits * in * out : 0) + bias_parts(n) * out) * sizeof(float);
}

namespace opal_head {
template <class T> __global__ __launch_bounds__(BLOCK) void col_sums_kernel(const T *x, uint64_t ld, uint64_t n, uint32_t cols, uint64_t rows, float *part)
{
    const uint32_t c = blockIdx.x * BLOCK + threadIdx.x;
    if (c >= cols) return;
    const uint64_t beg = blockIdx.y * rows, end = beg + rows < n ? beg + rows : n;
    float s = 0.f;
    for (uint64_t r = beg; r < end; r++) s += (float)x[r * ld + c];
    part[(uint64_t)blockIdx.y * cols + c] = s;
}

// out = the sum of the splits' matrices, in their order
__global__ __launch_bounds__(BLOCK) void sum_splits_kernel(const float *part, uint64_t splits, uint64_t each, uint32_t cols, float *out, uint64_t ld)
{
    for (uint64_t i = (uint64_t)blockIdx.x * BLOCK + threadIdx.x; i < each; i += (uint64_t)gridDim.x * BLOCK) {
        float s = part[i];
        for (uint64_t p = 1; p < splits; p++) s += part[p * each + i];
        out[i / cols * ld + i % cols] = s;
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
    OPAL_TRY(check_matrix(ctx, who, "dw", d_dw, OPAL_F32, lddw, out, in, true));
    if (!type_ok(type)) return bad_arg(ctx, who, "unknown element type");
    if (!d_dw && !d_dbias) return bad_arg(ctx, who, "neither dw nor dbias is asked for");
    const uint64_t need = opal_linear_grad_weight_workspace(n, in, out, type);
    if (need && (!d_work || work_bytes < need)) return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": the workspace is smaller than opal_linear_grad_weight_workspace says");
    if (reinterpret_cast<uintptr_t>(d_work) % 16) return bad_arg(ctx, who, "the workspace must be 16-byte aligned");
    OnDevice on(ctx->device);
    OPAL_HIP_CHECK(ctx, on.err);
    const Splits s = weight_splits(n, in, out, type);
    float *part = (float *)d_work;
    const uint64_t each = (uint64_t)in * out;
    if (d_dw) {
        Linear g{};
        g.a = (const char *)d_dy; g.lda = lddy; g.b = (const char *)d_x; g.ldb = ldx;
        g.M = out; g.N = in; g.K = n;
        const bool dma = aligned16(d_dy, lddy, type) && aligned16(d_x, ldx, type);
        const int tile = s.tile == 2 && !dma ? 1 : s.tile;
        if (tiles_of(out, in, tile) * s.splits >= (1ull << 31)) return opal::fail(ctx, OPAL_ERANGE, std::string(who) + ": in times out is too large for one call");
        set_tiles(g, tile);
        g.splits = (uint32_t)s.splits;
        g.items = g.tm * g.tn * g.splits;
        g.blocks = std::min<uint32_t>(g.items, ctx->num_cus);
        g.ksplit = s.rows;
        g.y = s.splits > 1 ? part : d_dw; g.y_type = OPAL_F32; g.ldy = s.splits > 1 ? in : lddw; g.y_split = each;
        OPAL_HIP_CHECK(ctx, launch(g, type, GWT, tile, dma, ctx->stream));
        if (s.splits > 1) {
            hipLaunchKernelGGL(sum_splits_kernel, dim3((unsigned)std::min<uint64_t>((each + BLOCK - 1) / BLOCK, 4096)), dim3(BLOCK), 0, ctx->stream, part, s.splits, each, in, d_dw, lddw);
            OPAL_HIP_CHECK(ctx, hipGetLastError());
        }
    }
    if (d_dbias) {
        float *bp = part + (s.splits > 1 ? s.splits * each : 0);
        const uint64_t parts = bias_parts(n);
        if (n) {
            const uint64_t rows = (n + parts - 1) / parts;
            const dim3 grid((out + BLOCK - 1) / BLOCK, (unsigned)parts);
            if (type == OPAL_F32) hipLaunchKernelGGL(col_sums_kernel<float>, grid, dim3(BLOCK), 0, ctx->stream, (const float *)d_dy, lddy, n, out, rows, bp);
            else if (type == OPAL_F16) hipLaunchKernelGGL(col_sums_kernel<f16_t>, grid, dim3(BLOCK), 0, ctx->stream, (const f16_t *)d_dy, lddy, n, out, rows, bp);
            else hipLaunchKernelGGL(col_sums_kernel<bf16_t>, grid, dim3(BLOCK), 0, ctx->stream, (const bf16_t *)d_dy, lddy, n, out, rows, bp);
            OPAL_HIP_CHECK(ctx, hipGetLastError());
        }
        sum_parts(bp, parts, out, out, d_dbias, ctx->stream);
        OPAL_HIP_CHECK(ctx, hipGetLastError());
    }
    return OPAL_OK;
}
