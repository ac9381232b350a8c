// Short causal convolution over the tokens of every channel, x [B][D][L], weights [D][W], W = 2..4:
//
//   v_t = b + sum_k w_k x_{t-W+1+k},   y_t = v_t or silu(v_t),   x_t for t < 0 is the state [B][D][W-1] (or zero)
//   backward, dv_t = dy_t silu'(v_t):
//   dx_t = sum_k w_k dv_{t+W-1-k},  dw_k = sum_t dv_t x_{t-W+1+k},  db = sum_t dv_t,  dstate = dx at t < 0
//
// Bound by HBM: 2 (forward) or 3 (backward) times the tensor.  A lane owns 8 consecutive tokens of one channel; the
// W-1 tokens before them (and, backward, after them) come from the cache with one more load each, and the pre-activation
// of the W-1 tokens after them is formed again: the slope there is another lane's.  64 lanes walk along a long row, 8
// lanes along a short one (so that a wave has 8 rows); a row of fewer than 8 tokens is one lane's.
// A row whose length is no multiple of 8 ends in a chunk that is pulled back to the row's end: its first tokens are
// stored twice with the same bits and left out of the weight's sums.
// 8 x 384 x 4096 bf16: 12 to 13 us forward (3.9 to 4.2 TB/s), 21 to 22 backward (3.5 TB/s, below the 4.8 of a copy: two loads more a tensor for the
// neighbours' tokens) and 3.9 for the sums of the weight's shares; a token, or a piece of a thousand, is a launch: 2 to 4 us.
#include "seq_common.hpp"

namespace rst {

constexpr int CC_TOK = 8;             // tokens of a lane
constexpr int CC_PART = 8;            // floats of a row's partial sums: dw[W], db, padding

template <typename T> struct ConvRow {
    const T* x; const T* state; int64_t L; int W;
    __device__ __forceinline__ float at(int64_t t) const {               // t >= -(W-1)
        if (t >= 0) return t < L ? Store<T>::get(x[t]) : 0.f;
        return state != nullptr ? Store<T>::get(state[t + W - 1]) : 0.f;
    }
};

__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }
__device__ __forceinline__ float silu_slope(float v) {
    const float s = sigmoid(v);
    return s * fmaf(v, 1.0f - s, 1.0f);
}

struct CausalConv {
    const void* x; const float* w; const float* b; const void* state_in;
    void* y; void* state_out;                                            // forward
    const void* dy; const void* dend; void* dx; void* dstate; float* partial;   // backward
    int B, D; int64_t L; int silu;
    int nchunk, nseg, per_seg;                                           // chunks of 8 tokens: in a row, segments, chunks of a segment
};

// the row and segment of this lane's group of TX lanes
template <int TX>
__device__ __forceinline__ bool conv_place(const CausalConv& a, int64_t* row, int* seg, int* lane) {
    uint32_t item = block_index<256>() * (256 / TX) + threadIdx.x / TX;         // rows x segments < 2^31: causal_conv_plan
    if (TX == 64) item = __builtin_amdgcn_readfirstlane(item);           // one row to a wave: its weights are scalar loads
    *lane = threadIdx.x % TX;
    *seg = (int)(item % (uint32_t)a.nseg);
    *row = item / (uint32_t)a.nseg;
    return *row < (int64_t)a.B * a.D;
}

template <typename T, int W, int TX>
__global__ void __launch_bounds__(256)
causal_conv_fwd_kernel(const CausalConv a) {
    int64_t row; int seg, lane;
    if (!conv_place<TX>(a, &row, &seg, &lane)) return;
    const int d = (int)((uint32_t)row % (uint32_t)a.D);
    float w[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = a.w[(int64_t)d * W + k];
    const float b = a.b != nullptr ? a.b[d] : 0.f;
    const ConvRow<T> in{static_cast<const T*>(a.x) + row * a.L,
                        a.state_in ? static_cast<const T*>(a.state_in) + row * (W - 1) : nullptr, a.L, W};
    T* y = static_cast<T*>(a.y) + row * a.L;
    T* end = a.state_out ? static_cast<T*>(a.state_out) + row * (W - 1) : nullptr;
    const int last = (seg + 1) * a.per_seg < a.nchunk ? (seg + 1) * a.per_seg : a.nchunk;
    for (int c = seg * a.per_seg + lane; c < last; c += TX) {
        const int64_t nat = (int64_t)c * CC_TOK;
        const int64_t s = nat + CC_TOK <= a.L ? nat : a.L - CC_TOK;
        float v[W - 1 + CC_TOK];
        Raw<T, CC_TOK> raw;
        raw.load(in.x + s);
        if (s >= 4) {
            Raw<T, 4> before;
            before.load(in.x + s - 4);
#pragma unroll
            for (int i = 0; i < W - 1; ++i) v[i] = before.get(4 - (W - 1) + i);
        } else {
#pragma unroll
            for (int i = 0; i < W - 1; ++i) v[i] = in.at(s - (W - 1) + i);
        }
#pragma unroll
        for (int i = 0; i < CC_TOK; ++i) v[W - 1 + i] = raw.get(i);
        float o[CC_TOK];
#pragma unroll
        for (int i = 0; i < CC_TOK; ++i) {
            float t = b;
#pragma unroll
            for (int k = 0; k < W; ++k) t = fmaf(w[k], v[i + k], t);
            o[i] = a.silu ? silu(t) : t;
        }
        Raw<T, CC_TOK> out;
        out.pack(o);
        out.store(y + s);
        if (end != nullptr && c == a.nchunk - 1) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) end[j] = Store<T>::put(v[CC_TOK + j]);
        }
    }
}

// a row of fewer than 8 tokens per lane
template <typename T, int W>
__global__ void __launch_bounds__(256)
causal_conv_fwd_short_kernel(const CausalConv a) {
    const int64_t row = (int64_t)block_index<256>() * 256 + threadIdx.x;
    if (row >= (int64_t)a.B * a.D) return;
    const int d = (int)(row % a.D), L = (int)a.L;
    const ConvRow<T> in{static_cast<const T*>(a.x) + row * a.L,
                        a.state_in ? static_cast<const T*>(a.state_in) + row * (W - 1) : nullptr, a.L, W};
    for (int t = 0; t < L; ++t) {
        float v = a.b != nullptr ? a.b[d] : 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) v = fmaf(a.w[(int64_t)d * W + k], in.at(t - W + 1 + k), v);
        static_cast<T*>(a.y)[row * a.L + t] = Store<T>::put(a.silu ? silu(v) : v);
    }
    if (a.state_out != nullptr)
        for (int j = 0; j < W - 1; ++j) static_cast<T*>(a.state_out)[row * (W - 1) + j] = Store<T>::put(in.at(L + j - (W - 1)));
}

template <typename T, int W, int TX>
__global__ void __launch_bounds__(256)
causal_conv_bwd_kernel(const CausalConv a) {
    int64_t row; int seg, lane;
    const bool live = conv_place<TX>(a, &row, &seg, &lane);
    if (TX == 64 && !live) return;                                       // (a whole wave; the groups of 8 share one below)
    if (!live) { row = 0; seg = 0; }
    const int d = (int)((uint32_t)row % (uint32_t)a.D);
    float w[W], pw[W], pb = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) { w[k] = a.w[(int64_t)d * W + k]; pw[k] = 0.f; }
    const float b = a.b != nullptr ? a.b[d] : 0.f;
    const ConvRow<T> in{static_cast<const T*>(a.x) + row * a.L,
                        a.state_in ? static_cast<const T*>(a.state_in) + row * (W - 1) : nullptr, a.L, W};
    const T* dy = static_cast<const T*>(a.dy) + row * a.L;
    T* dx = static_cast<T*>(a.dx) + row * a.L;
    const T* dend = a.dend ? static_cast<const T*>(a.dend) + row * (W - 1) : nullptr;
    const int last = !live ? 0 : (seg + 1) * a.per_seg < a.nchunk ? (seg + 1) * a.per_seg : a.nchunk;
    for (int c = seg * a.per_seg + lane; c < last; c += TX) {
        const int64_t nat = (int64_t)c * CC_TOK;
        const int64_t s = nat + CC_TOK <= a.L ? nat : a.L - CC_TOK;
        const int dup = (int)(nat - s);
        constexpr int N = CC_TOK + W - 1;                                // tokens whose slope is needed
        float v[N + W - 1], dv[N];
        Raw<T, CC_TOK> raw, rdy;
        raw.load(in.x + s);
        rdy.load(dy + s);
        if (s >= 4) {
            Raw<T, 4> before;
            before.load(in.x + s - 4);
#pragma unroll
            for (int i = 0; i < W - 1; ++i) v[i] = before.get(4 - (W - 1) + i);
        } else {
#pragma unroll
            for (int i = 0; i < W - 1; ++i) v[i] = in.at(s - (W - 1) + i);
        }
#pragma unroll
        for (int i = 0; i < CC_TOK; ++i) { v[W - 1 + i] = raw.get(i); dv[i] = rdy.get(i); }
        const int64_t e = s + CC_TOK;
        if (e + 4 <= a.L) {
            Raw<T, 4> ax, ad;
            ax.load(in.x + e);
            ad.load(dy + e);
#pragma unroll
            for (int i = 0; i < W - 1; ++i) { v[W - 1 + CC_TOK + i] = ax.get(i); dv[CC_TOK + i] = ad.get(i); }
        } else {
#pragma unroll
            for (int i = 0; i < W - 1; ++i) {
                v[W - 1 + CC_TOK + i] = in.at(e + i);
                dv[CC_TOK + i] = e + i < a.L ? Store<T>::get(dy[e + i]) : 0.f;
            }
        }
        if (a.silu) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float t = b;
#pragma unroll
                for (int k = 0; k < W; ++k) t = fmaf(w[k], v[i + k], t);
                dv[i] = i < CC_TOK || e + (i - CC_TOK) < a.L ? dv[i] * silu_slope(t) : 0.f;
            }
        }
        float o[CC_TOK];
#pragma unroll
        for (int i = 0; i < CC_TOK; ++i) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) t = fmaf(w[k], dv[i + W - 1 - k], t);
            o[i] = t;
            if (i >= dup) {
                pb += dv[i];
#pragma unroll
                for (int k = 0; k < W; ++k) pw[k] = fmaf(dv[i], v[i + k], pw[k]);
            }
        }
        if (dend != nullptr && e > a.L - (W - 1)) {                      // the last W-1 tokens are the final state too
#pragma unroll
            for (int i = 0; i < CC_TOK; ++i) {
                const int64_t j = s + i - (a.L - (W - 1));
                if (j >= 0) o[i] += Store<T>::get(dend[j]);
            }
        }
        Raw<T, CC_TOK> out;
        out.pack(o);
        out.store(dx + s);
        if (a.dstate != nullptr && c == 0) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                float t = 0.f;
#pragma unroll
                for (int k = 0; k <= j; ++k) t = fmaf(w[k], dv[j - k], t);
                static_cast<T*>(a.dstate)[row * (W - 1) + j] = Store<T>::put(t);
            }
        }
    }
#pragma unroll
    for (int off = TX / 2; off > 0; off >>= 1) {
        pb += __shfl_xor(pb, off, 64);
#pragma unroll
        for (int k = 0; k < W; ++k) pw[k] += __shfl_xor(pw[k], off, 64);
    }
    if (live && lane == 0) {
        float* p = a.partial + (((int64_t)((uint32_t)row / (uint32_t)a.D) * a.nseg + seg) * a.D + d) * CC_PART;
#pragma unroll
        for (int k = 0; k < W; ++k) p[k] = pw[k];
        p[W] = pb;
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(256)
causal_conv_bwd_short_kernel(const CausalConv a) {
    const int64_t row = (int64_t)block_index<256>() * 256 + threadIdx.x;
    if (row >= (int64_t)a.B * a.D) return;
    const int d = (int)(row % a.D), L = (int)a.L;
    const ConvRow<T> in{static_cast<const T*>(a.x) + row * a.L,
                        a.state_in ? static_cast<const T*>(a.state_in) + row * (W - 1) : nullptr, a.L, W};
    float w[W], pw[W], pb = 0.f, dv[CC_TOK + W - 1], dfull[CC_TOK + W - 1];
#pragma unroll
    for (int k = 0; k < W; ++k) { w[k] = a.w[(int64_t)d * W + k]; pw[k] = 0.f; }
    const float b = a.b != nullptr ? a.b[d] : 0.f;
#pragma unroll
    for (int i = 0; i < CC_TOK + W - 1; ++i) { dv[i] = 0.f; dfull[i] = 0.f; }
#pragma unroll
    for (int t = 0; t < CC_TOK - 1; ++t) {
        if (t < L) {
            float v = b;
#pragma unroll
            for (int k = 0; k < W; ++k) v = fmaf(w[k], in.at(t - W + 1 + k), v);
            dv[t] = Store<T>::get(static_cast<const T*>(a.dy)[row * a.L + t]) * (a.silu ? silu_slope(v) : 1.f);
            pb += dv[t];
#pragma unroll
            for (int k = 0; k < W; ++k) {
                pw[k] = fmaf(dv[t], in.at(t - W + 1 + k), pw[k]);
                dfull[t + k] = fmaf(w[k], dv[t], dfull[t + k]);           // position p = t + W - 1 of the state and the row
            }
        }
    }
#pragma unroll
    for (int p = 0; p < CC_TOK - 1 + W - 1; ++p) {
        if (p < L + W - 1) {
            float v = dfull[p];
            if (a.dend != nullptr && p >= L) v += Store<T>::get(static_cast<const T*>(a.dend)[row * (W - 1) + p - L]);
            if (p >= W - 1) static_cast<T*>(a.dx)[row * a.L + p - (W - 1)] = Store<T>::put(v);
            else if (a.dstate != nullptr) static_cast<T*>(a.dstate)[row * (W - 1) + p] = Store<T>::put(v);
        }
    }
    float* p = a.partial + row * CC_PART;
#pragma unroll
    for (int k = 0; k < W; ++k) p[k] = pw[k];
    p[W] = pb;
}

// dw[d][k], db[d]: the partial sums of all samples and segments in a fixed order, a block per channel
template <int W>
__global__ void __launch_bounds__(256)
causal_conv_reduce_kernel(const float* __restrict__ partial, int n, int D, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float red[32][CC_PART + 1];
    const int d = (int)block_index<256>(), k = threadIdx.x % CC_PART, slice = threadIdx.x / CC_PART;
    float s = 0.f;
    if (d >= D) return;
    if (k <= W)
        for (int64_t p = slice; p < n; p += 32) s += partial[(p * D + d) * CC_PART + k];
    red[slice][k] = s;
    __syncthreads();
    for (int h = 16; h > 0; h >>= 1) {
        if (slice < h) red[slice][k] += red[slice + h][k];
        __syncthreads();
    }
    if (slice == 0) {
        if (k < W) dw[(int64_t)d * W + k] = red[0][k];
        else if (k == W && db != nullptr) db[d] = red[0][k];
    }
}

// one token: y = act(b + w . [state, x]), the state moves on by one.  state_out may be the state itself.
template <typename T, int W>
__global__ void __launch_bounds__(256)
causal_conv_update_kernel(const T* __restrict__ x, const T* state, T* state_out, const float* __restrict__ w,
                          const float* __restrict__ b, T* __restrict__ y, int64_t n, int D, int act) {
    const int64_t i = (int64_t)block_index<256>() * 256 + threadIdx.x;
    if (i >= n) return;
    const int d = (int)(i % D);
    T in[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) in[k] = state[i * (W - 1) + k];
    in[W - 1] = x[i];
    float v = b != nullptr ? b[d] : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) v = fmaf(w[(int64_t)d * W + k], Store<T>::get(in[k]), v);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) state_out[i * (W - 1) + k] = in[k + 1];
    y[i] = Store<T>::put(act ? silu(v) : v);
}

// 64 lanes to a row of more than 256 tokens, 8 to a shorter one: 64 x 384 rows of 256 fp32 tokens take 13 us forward and 21
// backward with 8, 15 and 26 with 64; 16 x 256 rows of 384 bf16 tokens 7.9 and 14.9 with 8, 6.6 and 10.7 with 64.  A long row is
// cut into segments where there are too few rows for 8192 waves (8 a SIMD): 192 rows of 16384 bf16 tokens 19 and 44 us
// uncut, 7.6 and 12 so.
static int causal_conv_plan(CausalConv* a) {
    a->nchunk = (int)cdiv(a->L, CC_TOK);
    const int64_t rows = (int64_t)a->B * a->D;
    a->nseg = 1;
    int tx = 8;
    if (a->nchunk > 32) {
        tx = 64;
        const int64_t most = cdiv(a->nchunk, 64), want = cdiv(8192, rows);
        a->nseg = (int)(want < most ? want : most);
    }
    a->per_seg = (int)round_up(cdiv(a->nchunk, a->nseg), 64);
    a->nseg = (int)cdiv(a->nchunk, a->per_seg);
    return tx;
}

template <typename T, int W>
static int causal_conv_fwd_t(CausalConv a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.D;
    ProfScope prof(st, "causal_conv_fwd", (2.0 * W + 5) * rows * a.L, 2.0 * sizeof(T) * rows * a.L);
    if (a.L < CC_TOK) {
        hipLaunchKernelGGL((causal_conv_fwd_short_kernel<T, W>), grid_of<256>(cdiv(rows, 256)), dim3(256), 0, st, a);
    } else if (causal_conv_plan(&a) == 64) {
        hipLaunchKernelGGL((causal_conv_fwd_kernel<T, W, 64>), grid_of<256>(cdiv(rows * a.nseg, 4)), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((causal_conv_fwd_kernel<T, W, 8>), grid_of<256>(cdiv(rows, 32)), dim3(256), 0, st, a);
    }
    RST_LAUNCH_CHECK();
    return RST_OK;
}

template <typename T, int W>
static int causal_conv_bwd_t(CausalConv a, float* dw, float* db, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.D;
    ProfScope prof(st, "causal_conv_bwd", (6.0 * W + 10) * rows * a.L, 3.0 * sizeof(T) * rows * a.L);
    if (a.L < CC_TOK) {
        a.nseg = 1;
        hipLaunchKernelGGL((causal_conv_bwd_short_kernel<T, W>), grid_of<256>(cdiv(rows, 256)), dim3(256), 0, st, a);
    } else if (causal_conv_plan(&a) == 64) {
        hipLaunchKernelGGL((causal_conv_bwd_kernel<T, W, 64>), grid_of<256>(cdiv(rows * a.nseg, 4)), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((causal_conv_bwd_kernel<T, W, 8>), grid_of<256>(cdiv(rows, 32)), dim3(256), 0, st, a);
    }
    RST_LAUNCH_CHECK();
    hipLaunchKernelGGL((causal_conv_reduce_kernel<W>), grid_of<256>(a.D), dim3(256), 0, st, a.partial, a.B * a.nseg, a.D, dw, db);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

template <typename T, int W>
static int causal_conv_update_t(const T* x, const T* state, T* state_out, const float* w, const float* b, T* y, int64_t n, int D, int act,
                                hipStream_t st) {
    ProfScope prof(st, "causal_conv_update", (2.0 * W + 5) * n, 2.0 * W * sizeof(T) * n);
    hipLaunchKernelGGL((causal_conv_update_kernel<T, W>), grid_of<256>(cdiv(n, 256)), dim3(256), 0, st, x, state, state_out, w, b, y, n,
                       D, act);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

static size_t causal_conv_bwd_ws(int B, int D, int64_t L) {
    CausalConv a{};
    a.B = B; a.D = D; a.L = L; a.nseg = 1;
    if (L >= CC_TOK) causal_conv_plan(&a);
    return (size_t)B * a.nseg * D * CC_PART * sizeof(float);
}

static int causal_conv_check(const char* what, int dtype, int B, int D, int64_t L, int W) {
    RST_REQUIRE(dtype == RST_DTYPE_F32 || dtype == RST_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
    RST_REQUIRE(B > 0 && D > 0 && L > 0, "%s: empty shape B=%d D=%d L=%lld", what, B, D, (long long)L);
    RST_REQUIRE(W >= 2 && W <= 4, "%s: width %d (2, 3 or 4)", what, W);
    RST_REQUIRE((int64_t)B * D <= (1ll << 30) && L <= (1ll << 31), "%s: shape out of range B=%d D=%d L=%lld", what, B, D, (long long)L);
    return RST_OK;
}

}  // namespace rst

using namespace rst;

#define CC_WIDTHS(CALL, T)                                                                                              \
    (W == 2 ? CALL(T, 2) : W == 3 ? CALL(T, 3) : CALL(T, 4))
#define CC_TYPES(CALL) (dtype == RST_DTYPE_F32 ? CC_WIDTHS(CALL, float) : CC_WIDTHS(CALL, bf16_t))

extern "C" {

int rst_causal_conv1d_fwd(const void* x, int32_t dtype, const float* weight, const float* bias, const void* state_in, void* y,
                          void* state_out, int32_t B, int32_t D, int64_t L, int32_t W, int32_t silu, void* stream) {
    RST_REQUIRE(x && weight && y, "causal_conv1d_fwd: null operand");
    RST_TRY(causal_conv_check("causal_conv1d_fwd", dtype, B, D, L, W));
    CausalConv a{};
    a.x = x; a.w = weight; a.b = bias; a.state_in = state_in; a.y = y; a.state_out = state_out;
    a.B = B; a.D = D; a.L = L; a.silu = silu;
    hipStream_t st = static_cast<hipStream_t>(stream);
#define FWD(T, W_) causal_conv_fwd_t<T, W_>(a, st)
    return CC_TYPES(FWD);
#undef FWD
}

size_t rst_causal_conv1d_bwd_workspace_bytes(int32_t B, int32_t D, int64_t L) {
    if (causal_conv_check("causal_conv1d_bwd_workspace_bytes", RST_DTYPE_F32, B, D, L, 2) != RST_OK) return 0;
    return causal_conv_bwd_ws(B, D, L);
}

int rst_causal_conv1d_bwd(const void* x, int32_t dtype, const float* weight, const float* bias, const void* state_in,
                          const void* dy, const void* dstate_out, void* dx, float* dweight, float* dbias, void* dstate_in,
                          int32_t B, int32_t D, int64_t L, int32_t W, int32_t silu, void* workspace, size_t workspace_bytes,
                          void* stream) {
    RST_REQUIRE(x && weight && dy && dx && dweight, "causal_conv1d_bwd: null operand");
    RST_TRY(causal_conv_check("causal_conv1d_bwd", dtype, B, D, L, W));
    if (workspace == nullptr || workspace_bytes < causal_conv_bwd_ws(B, D, L))
        return fail(RST_ERR_WORKSPACE, "causal_conv1d_bwd: workspace too small (%zu < %zu)", workspace_bytes, causal_conv_bwd_ws(B, D, L));
    CausalConv a{};
    a.x = x; a.w = weight; a.b = bias; a.state_in = state_in; a.dy = dy; a.dend = dstate_out; a.dx = dx; a.dstate = dstate_in;
    a.partial = static_cast<float*>(workspace);
    a.B = B; a.D = D; a.L = L; a.silu = silu;
    hipStream_t st = static_cast<hipStream_t>(stream);
#define BWD(T, W_) causal_conv_bwd_t<T, W_>(a, dweight, dbias, st)
    return CC_TYPES(BWD);
#undef BWD
}

int rst_causal_conv1d_update(const void* x, int32_t dtype, const void* state_in, void* state_out, const float* weight,
                             const float* bias, void* y, int32_t B, int32_t D, int32_t W, int32_t silu, void* stream) {
    RST_REQUIRE(x && state_in && state_out && weight && y, "causal_conv1d_update: null operand");
    RST_TRY(causal_conv_check("causal_conv1d_update", dtype, B, D, 1, W));
    const int64_t n = (int64_t)B * D;
    hipStream_t st = static_cast<hipStream_t>(stream);
#define UPD(T, W_)                                                                                                      \
    causal_conv_update_t<T, W_>(static_cast<const T*>(x), static_cast<const T*>(state_in), static_cast<T*>(state_out), weight, bias, \
                                static_cast<T*>(y), n, D, silu, st)
    return CC_TYPES(UPD);
#undef UPD
}

}  // extern "C"
