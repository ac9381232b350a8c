// Layer norm of token rows: x [rows][C], C contiguous, fp32 or bf16 storage, fp32 statistics and parameters.
//
//   mu = mean x, v = mean (x - mu)^2, r = 1 / sqrt(v + eps)
//   with bias:  y = (x - mu) r w + b        bias-free:  y = x r w        (the two norms of model/Restromer.py:28-61)
//   backward, g = dy w, xh = (x - mu) r:
//   with bias:  dx = r (g - mean g - xh mean(g xh)),            dw = sum_rows dy xh,    db = sum_rows dy
//   bias-free:  dx = r g - r^2 xh mean(g x),                    dw = sum_rows dy x r
//
// The channel norm of layernorm.hip has lanes over pixels; here a row is contiguous, so LPR lanes share a row, each
// holding NV vectors of 16 bytes of it in registers: x (and dy) are read once, the two statistics are two butterfly
// sums over the LPR lanes.  Bound by HBM: 2 (forward) or 3 (backward) times the tensor.
//
// The mean is summed relative to the row's first value: of a flat row every difference is an exact zero, so its mean is its
// value and its variance zero.  (The sum of the values themselves is a rounded one: 96 values of 1000.1 fp32 came to a mean
// 6e-5 off, which 1 / sqrt(eps) makes 0.02 of.)  A row's own spread bounds the differences' roundings in any case.
// Half the differences, each over C, are added up, so that no row of finite values overflows here.
//
// A row whose length is no multiple of the vector ends in a vector that is pulled back to the row's end: its first
// values are the neighbour's last ones again, left out of every sum and stored twice with the same bits.
// Forward 134 us for 1048576 x 96 fp32 (6.0 TB/s), 12 to 14 us for 131072 x 96 bf16 (3.6 to 4.2 TB/s: launch and fill count there),
// 3.6 us, a launch, for 64 x 384.
#include "seq_common.hpp"

namespace rst {

// where vector j of a lane starts in the row, and how many of its first values belong to another lane's: all of them
// where the row has no such vector (the lane reads the row's start again, so that no load is behind a branch)
template <int VEC>
__device__ __forceinline__ void row_vec(int j, int C, int* start, int* dup) {
    const int nat = j * VEC;
    *start = nat + VEC <= C ? nat : nat < C ? C - VEC : 0;
    *dup = nat < C ? nat - *start : VEC;
}

// sum over the LPR lanes of a row; LPR = 256: over the block, through `red` (4 floats)
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    constexpr int IN_WAVE = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int off = IN_WAVE / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (LPR == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0] + red[1] + red[2] + red[3];
    }
    return v;
}

template <typename T, int VEC, int LPR, int NV>
__global__ void __launch_bounds__(256)
norm_rows_fwd_kernel(const T* __restrict__ x, const float* __restrict__ weight, const float* __restrict__ bias,
                     T* __restrict__ y, int64_t rows, int C, float eps) {
    __shared__ float red[4];
    const int lane = threadIdx.x % LPR;
    const int64_t row = (int64_t)block_index<256>() * (256 / LPR) + threadIdx.x / LPR;
    const bool live = row < rows;
    const T* xr = x + (live ? row : 0) * C;
    Raw<T, VEC> raw[NV];
    int start[NV], dup[NV];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        row_vec<VEC>(lane + j * LPR, C, &start[j], &dup[j]);
        raw[j].load(xr + start[j]);
    }
    const float first = Store<T>::get(xr[0]), invC = 1.0f / (float)C;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s = fmaf(i >= dup[j] ? fmaf(0.5f, raw[j].get(i), -0.5f * first) : 0.f, invC, s);
    const float mu = fmaf(2.0f, row_sum<LPR>(s, red), first);
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float d = i >= dup[j] ? raw[j].get(i) - mu : 0.f;
            q = fmaf(d, d, q);
        }
    const float r = 1.0f / sqrtf(row_sum<LPR>(q, red) * invC + eps);
    if (!live) return;
    T* yr = y + row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (dup[j] < VEC) {
            Raw<float, VEC> w;
            w.load(weight + start[j]);
            float o[VEC];
            if (bias != nullptr) {
                Raw<float, VEC> b;
                b.load(bias + start[j]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = fmaf((raw[j].get(i) - mu) * r, w.get(i), b.get(i));
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = raw[j].get(i) * r * w.get(i);
            }
            raw[j].pack(o);
            raw[j].store(yr + start[j]);
        }
}

// Blocks walk over the rows, the next row's values on the way (448 -> 240 us for 1048576 x 96 fp32: 5.0 TB/s; 131072 x 96 bf16:
// 21 us, 3.6 TB/s); a lane keeps the sums of dw and db of its own columns in registers, the block adds those of its row
// groups through LDS and writes one row of partial sums [2][C]; norm_rows_reduce_kernel adds the blocks' rows in a fixed order
// (the same bits run to run; 4 to 5 us).
template <typename T, int VEC, int LPR, int NV>
__global__ void __launch_bounds__(256, NV * VEC <= 12 ? 4 : NV * VEC <= 16 ? 3 : NV * VEC <= 24 ? 2 : 1)
norm_rows_bwd_kernel(const T* __restrict__ x, const float* __restrict__ weight, int with_bias, const T* __restrict__ dy,
                     T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int C, float eps) {
    constexpr int RPB = 256 / LPR;
    __shared__ float red[4];
    extern __shared__ __attribute__((aligned(16))) float acc[];            // [row groups][C], at most 32 KiB
    const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    int start[NV], dup[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) row_vec<VEC>(lane + j * LPR, C, &start[j], &dup[j]);
    float pw[NV][VEC], pb[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) { pw[j][i] = 0.f; pb[j][i] = 0.f; }
    const float invC = 1.0f / (float)C;

    const int64_t step = (int64_t)gridDim.x * RPB;
    Raw<T, VEC> rx[NV], rd[NV], nx[NV], nd[NV];
    T nfirst;
    auto fetch = [&](int64_t row0) {                                       // the next row is on its way while one is worked on
        const int64_t row = row0 + grp, base = (row < rows ? row : rows - 1) * C;
        nfirst = x[base];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            nx[j].load(x + base + start[j]);
            nd[j].load(dy + base + start[j]);
        }
    };
    fetch((int64_t)blockIdx.x * RPB);
    for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < rows; row0 += step) {
        const int64_t row = row0 + grp;
        const bool live = row < rows;
        const int64_t base = row * C;
#pragma unroll
        for (int j = 0; j < NV; ++j) { rx[j] = nx[j]; rd[j] = nd[j]; }
        const float first = Store<T>::get(nfirst);
        if (row0 + step < rows) fetch(row0 + step);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s = fmaf(i >= dup[j] ? fmaf(0.5f, rx[j].get(i), -0.5f * first) : 0.f, invC, s);
        const float mu = fmaf(2.0f, row_sum<LPR>(s, red), first);
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = i >= dup[j] ? rx[j].get(i) - mu : 0.f;
                q = fmaf(d, d, q);
            }
        const float r = 1.0f / sqrtf(row_sum<LPR>(q, red) * invC + eps);
        const float shift = with_bias ? 0.f : mu * r;                       // x r = xh + mu r
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Raw<float, VEC> w;
            w.load(weight + start[j]);
            const int own = live ? dup[j] : VEC;                            // a row past the last one adds nothing
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xh = (rx[j].get(i) - mu) * r, d = i >= own ? rd[j].get(i) : 0.f, g = d * w.get(i);
                s1 += g;
                s2 = fmaf(g, xh, s2);
                pw[j][i] = fmaf(d, xh + shift, pw[j][i]);
                pb[j][i] += d;
            }
        }
        s1 = row_sum<LPR>(s1, red);
        s2 = row_sum<LPR>(s2, red);
        // bias-free: mean(g x) = (s2 / r + mu s1) / C, and the factor r^2 turns it into r (s2 + mu r s1) / C
        const float k1 = with_bias ? s1 * invC : 0.f;
        const float k2 = with_bias ? s2 * invC : (s2 + shift * s1) * invC;
        if (live) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (dup[j] < VEC) {
                    Raw<float, VEC> w;
                    w.load(weight + start[j]);
                    float o[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float xh = (rx[j].get(i) - mu) * r;
                        o[i] = r * (fmaf(rd[j].get(i), w.get(i), -k1) - xh * k2);
                    }
                    rx[j].pack(o);
                    rx[j].store(dx + base + start[j]);
                }
        }
    }
    // the block's row groups: every one writes its sums to a row of LDS (a column belongs to one lane of a group), then a
    // thread adds up a column, in a fixed order
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (half == 1 && !with_bias) break;
        if (half) __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i >= dup[j]) acc[grp * C + start[j] + i] = half ? pb[j][i] : pw[j][i];
        __syncthreads();
        float* out = partial + ((int64_t)blockIdx.x * 2 + half) * C;
        for (int c = threadIdx.x; c < C; c += 256) {
            float v = 0.f;
#pragma unroll 4
            for (int g = 0; g < RPB; ++g) v += acc[g * C + c];
            out[c] = v;
        }
    }
}

// out[c] = sum over the partial rows, in a fixed order; 16 columns x 64 slices per block
__global__ void __launch_bounds__(1024)
norm_rows_reduce_kernel(const float* __restrict__ partial, int n, int C, float* __restrict__ dweight, float* __restrict__ dbias) {
    __shared__ float red[64][17];
    const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const int half = blockIdx.y;
    const int c = blockIdx.x * 16 + col;
    float s = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int p = slice; p < n; p += 64) s += partial[((int64_t)p * 2 + half) * C + c];
    }
    red[slice][col] = s;
    __syncthreads();
    for (int w = 32; w > 0; w >>= 1) {
        if (slice < w) red[slice][col] += red[slice + w][col];
        __syncthreads();
    }
    if (slice == 0 && c < C) (half ? dbias : dweight)[c] = red[0][col];
}

constexpr int NR_MAX_C = 8192;
constexpr int NR_BWD_BLOCKS = 1024;           // four blocks on each of the 256 compute units

struct NormRowsPlan { int vec, lpr, nv; };
// Lanes per row and vectors per lane: the pair that leaves the fewest lanes without a vector, the fewer lanes (the
// shorter butterfly) where two are alike.  Against one vector a lane, the next power of two of them, forward: 1048576 x 96
// fp32 136 to 205 us, 262144 x 192 bf16 37 to 47, 262144 x 130 bf16 29 to 40, 262144 x 48 fp32 20.4 to 21.7.  A lane holds at
// most 24 values of a bf16 row: 32 take all 256 registers.
// Rows beyond 64 lanes (1536 values bf16, 1024 fp32) go to the 256 lanes of a block with 2, 4 or 8 vectors, where up to half of the
// vectors are idle and the backward kernel spills with 4 fp32 vectors (26 registers).  For 2^28 values bf16 (2^27 fp32) the
// forward kernel reaches 5.6 to 5.9 TB/s at 512 to 1536 values a row and the backward kernel 4.8 to 5.0; with 256 lanes bf16 rows of
// 1600, 2048 and 4096 values come to 3.7, 4.4 and 4.9 forward and 1.9, 2.4 and 3.6 backward, fp32 rows of 2048, 2500, 4096 and 8192
// to 5.8, 5.3, 5.4 and 5.5 forward and 5.0, 1.8, 2.4 and 4.1 backward.
static NormRowsPlan norm_rows_plan(int C, int full_vec) {
    const int most = full_vec == 8 ? 3 : 4;
    NormRowsPlan p{full_vec, 0, 0};
    if (C < full_vec) p.vec = 1;
    const int n = (int)cdiv(C, p.vec);
    int best = 1 << 30;
    for (int lpr = 8; lpr <= 64; lpr *= 2)
        for (int nv = 1; nv <= most; ++nv)
            if (lpr * nv >= n && lpr * nv < best) { best = lpr * nv; p.lpr = lpr; p.nv = nv; }
    if (p.lpr == 0) {
        p.lpr = 256;
        p.nv = n <= 512 ? 2 : n <= 1024 ? 4 : 8;
    }
    return p;
}

// blocks of the backward kernel, each with a row of partial sums [2][C]
static int64_t norm_rows_bwd_grid(int64_t rows, int lpr) {
    const int64_t want = cdiv(rows, 256 / lpr);
    return want < NR_BWD_BLOCKS ? want : NR_BWD_BLOCKS;
}
static size_t norm_rows_bwd_ws_bytes(int64_t rows, int C) {
    // (of the two types' plans the one with more blocks: the size is asked for without a type)
    const int64_t a = norm_rows_bwd_grid(rows, norm_rows_plan(C, Store<float>::VEC).lpr);
    const int64_t b = norm_rows_bwd_grid(rows, norm_rows_plan(C, Store<bf16_t>::VEC).lpr);
    return (size_t)(a > b ? a : b) * 2 * (size_t)C * sizeof(float);
}

// The pairs that the plan comes to for some length, fp32 (4 values a vector) or bf16 (8)
static constexpr bool nr_reached(int vec, int lpr, int nv) {
    if (lpr == 256) return 256 * nv * vec <= NR_MAX_C;
    if (lpr == 8) return nv <= (vec == 8 ? 3 : 4);
    return vec == 8 ? nv == 2 || nv == 3 : nv == 3 || nv == 4;
}
#define NR_CASES(X, ...)                                                                                                 \
    X(8, 1, __VA_ARGS__) X(8, 2, __VA_ARGS__) X(8, 3, __VA_ARGS__) X(8, 4, __VA_ARGS__) X(16, 2, __VA_ARGS__)              \
    X(16, 3, __VA_ARGS__) X(16, 4, __VA_ARGS__) X(32, 2, __VA_ARGS__) X(32, 3, __VA_ARGS__) X(32, 4, __VA_ARGS__)          \
    X(64, 2, __VA_ARGS__) X(64, 3, __VA_ARGS__) X(64, 4, __VA_ARGS__) X(256, 2, __VA_ARGS__) X(256, 4, __VA_ARGS__)        \
    X(256, 8, __VA_ARGS__)

// The kernel for a plan: every length of a row has exactly one.
#define NR_DISPATCH(KERNEL, LDS, GRID, ...)                                                                               \
    do {                                                                                                                \
        if (p.vec == 1) {                                                                                                 \
            hipLaunchKernelGGL((KERNEL<T, 1, 8, 1>), grid_of<256>(GRID), dim3(256), LDS, st, __VA_ARGS__);             \
        } else switch (p.lpr * 16 + p.nv) {                                                                              \
            NR_CASES(NR_CASE_OF, KERNEL, LDS, GRID, __VA_ARGS__)                                                          \
            default: return fail(RST_ERR_INVALID, "rows_norm: no kernel for C=%d", C);                                    \
        }                                                                                                               \
        RST_LAUNCH_CHECK();                                                                                              \
    } while (0)
#define NR_CASE_OF(L_, N_, KERNEL, LDS, GRID, ...)                                                                        \
    case L_ * 16 + N_:                                                                                                   \
        if constexpr (nr_reached(V, L_, N_))                                                                         \
            hipLaunchKernelGGL((KERNEL<T, V, L_, N_>), grid_of<256>(GRID), dim3(256), LDS, st, __VA_ARGS__);          \
        break;

template <typename T>
static int norm_rows_fwd_t(const T* x, const float* w, const float* b, T* y, int64_t rows, int C, float eps, hipStream_t st) {
    constexpr int V = Store<T>::VEC;
    const NormRowsPlan p = norm_rows_plan(C, V);
    const int64_t grid = cdiv(rows, 256 / p.lpr);
    RST_REQUIRE(grid < (1ll << 31), "rows_norm: %lld rows are out of range", (long long)rows);
    ProfScope prof(st, "rows_norm_fwd", 8.0 * rows * C, 2.0 * sizeof(T) * rows * C);
    NR_DISPATCH(norm_rows_fwd_kernel, 0, grid, x, w, b, y, rows, C, eps);
    return RST_OK;
}

template <typename T>
static int norm_rows_bwd_t(const T* x, const float* w, int with_bias, const T* dy, T* dx, float* dweight, float* dbias,
                           int64_t rows, int C, float eps, float* partial, hipStream_t st) {
    constexpr int V = Store<T>::VEC;
    const NormRowsPlan p = norm_rows_plan(C, V);
    const int grid = (int)norm_rows_bwd_grid(rows, p.lpr);
    ProfScope prof(st, "rows_norm_bwd", 14.0 * rows * C, 3.0 * sizeof(T) * rows * C);
    NR_DISPATCH(norm_rows_bwd_kernel, (size_t)(256 / p.lpr) * C * sizeof(float), grid, x, w, with_bias, dy, dx, partial, rows, C, eps);
    hipLaunchKernelGGL(norm_rows_reduce_kernel, dim3((unsigned)cdiv(C, 16), with_bias ? 2 : 1), dim3(1024), 0, st, partial, grid, C,
                       dweight, dbias);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

}  // namespace rst

using namespace rst;

extern "C" {

static int norm_rows_check(const char* what, int dtype, int64_t rows, int C, float eps) {
    RST_REQUIRE(dtype == RST_DTYPE_F32 || dtype == RST_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
    RST_REQUIRE(rows > 0 && C > 0 && rows <= (1ll << 40), "%s: empty shape or too many rows: rows=%lld C=%d", what, (long long)rows, C);
    RST_REQUIRE(C <= NR_MAX_C, "%s: C=%d too large (max %d)", what, C, NR_MAX_C);
    RST_REQUIRE(eps >= 0.f, "%s: eps=%g is negative or no number", what, (double)eps);
    return RST_OK;
}

int rst_rows_norm_fwd(const void* x, int32_t dtype, const float* weight, const float* bias, void* y, int64_t rows, int32_t C,
                      float eps, void* stream) {
    RST_REQUIRE(x && weight && y, "rows_norm_fwd: null operand");
    RST_TRY(norm_rows_check("rows_norm_fwd", dtype, rows, C, eps));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == RST_DTYPE_F32)
        return norm_rows_fwd_t(static_cast<const float*>(x), weight, bias, static_cast<float*>(y), rows, C, eps, st);
    return norm_rows_fwd_t(static_cast<const bf16_t*>(x), weight, bias, static_cast<bf16_t*>(y), rows, C, eps, st);
}

size_t rst_rows_norm_bwd_workspace_bytes(int64_t rows, int32_t C) {
    return rows > 0 && C > 0 && C <= NR_MAX_C ? norm_rows_bwd_ws_bytes(rows, C) : 0;
}

int rst_rows_norm_bwd(const void* x, int32_t dtype, const float* weight, int32_t with_bias, const void* dy, void* dx,
                      float* dweight, float* dbias, int64_t rows, int32_t C, float eps, void* workspace, size_t workspace_bytes,
                      void* stream) {
    RST_REQUIRE(x && weight && dy && dx && dweight, "rows_norm_bwd: null operand");
    RST_REQUIRE(!with_bias || dbias, "rows_norm_bwd: with_bias set but dbias is null");
    RST_TRY(norm_rows_check("rows_norm_bwd", dtype, rows, C, eps));
    if (workspace == nullptr || workspace_bytes < norm_rows_bwd_ws_bytes(rows, C))
        return fail(RST_ERR_WORKSPACE, "rows_norm_bwd: workspace too small (%zu < %zu)", workspace_bytes, norm_rows_bwd_ws_bytes(rows, C));
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* partial = static_cast<float*>(workspace);
    if (dtype == RST_DTYPE_F32)
        return norm_rows_bwd_t(static_cast<const float*>(x), weight, with_bias, static_cast<const float*>(dy), static_cast<float*>(dx),
                               dweight, dbias, rows, C, eps, partial, st);
    return norm_rows_bwd_t(static_cast<const bf16_t*>(x), weight, with_bias, static_cast<const bf16_t*>(dy), static_cast<bf16_t*>(dx),
                           dweight, dbias, rows, C, eps, partial, st);
}

}  // extern "C"
