// Selective state space scan over the tokens of every channel (x, delta, z, y: [B][D][L]; A: [D][N]; B, C: [B][G][N][L],
// channel d reads group d / (D/G)), its backward pass, and its form for one token.
//
//   dt = softplus(delta + bias),  a_t[n] = exp(dt_t A[n]),  h_t[n] = a_t[n] h_{t-1}[n] + dt_t x_t B_t[n]
//   s_t = sum_n C_t[n] h_t[n] + D x_t,   y_t = s_t or s_t silu(z_t)
//   backward, e_t = dy_t silu(z_t):  g_t[n] = C_t[n] e_t + a_{t+1}[n] g_{t+1}[n]   (from the last token to the first)
//   dC_t[n] = sum_d h e,  dB_t[n] = sum_d g dt x,  dx = dt sum_n g B + D e,  ddt = x sum_n g B + sum_n A a g h_{t-1},
//   dA[n] = sum_{b,t} dt a g h_{t-1},  dD = sum e x,  ddelta = ddt sigmoid(delta + bias),  dz = dy s silu'(z)
//
// Bound by the vector pipe and its waits, not by memory: one exponential and five more operations per state and token forward (16
// states: 96 operations for the 6 to 12 bytes of a bf16 or fp32 token), so the layout serves the instruction stream:
//   - a lane is a channel and holds four of its states; the waves of a block hold the other states of the same 64
//     channels.  B and C are then the same for a whole wave: one register holds its share of a tile and is the broadcast
//     operand of the matrix instruction that adds a token's input to 64 x 4 states (rank_one); LDS has it for the sums.
//   - tokens go in tiles of 16.  The tensors are token-contiguous, so a thread loads 4 tokens of one channel (a wave: 16
//     channels x 16 tokens), takes softplus once, and hands dt and dt x over through LDS, turned to lane = channel; the
//     waves' shares of s come back the same way.
//   - where there are too few channels to fill the chip, the tokens are cut into chunks: a first kernel takes every
//     chunk's own end state and the sum of its dt (its decay is exp(A sum dt)), and a chunk starts from the combination
//     of those before it.  That costs the exponentials a second time, so it is done only then (scan_plan).
//   - backward, a wave forms the tile's 16 x 4 states again from the state at the tile's start (kept by the forward
//     pass), holds them and the decays in registers, and walks back.
// State, decay, sums and partial sums are fp32.
#include "seq_common.hpp"

#include <utility>

namespace rst {

constexpr int ST = 16;                 // tokens of a tile
constexpr int SC = 64;                 // channels of a block
constexpr int SROW = 68;               // LDS row of a token: 64 channels and four more, so that 4 tokens apart is 16 banks apart

struct Scan {
    const void *x, *delta, *Bm, *Cm, *z, *dy;
    const float *A, *Dskip, *dbias, *h0, *dlast;
    void *y, *dx, *ddelta, *dB, *dC, *dz;
    float *last, *dh0;
    float* ckpt;                        // [B][tiles][4 W][D]: the state at every tile's start, or null
    float* cst;                         // [B][chunks][4 W][D]: what a chunk adds to the state behind (backward: before) it
    float* cdt;                         // [B][chunks][D]: sum of dt
    float* bcpart;                      // [channel blocks of a group][B][G][tiles * 2][W][64]: shares of dB and dC (tokens_fold)
    float* dApart;                      // [B][chunks][4 W][D]
    float* dDpart;                      // [B][chunks][2][D]: dD, dbias
    int B, D, G, N, Dg, cb;             // cb: channel blocks of a group
    int64_t L;
    int tiles, nchunk, per_chunk;       // per_chunk: tiles
    int softplus;
};

// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v|.  w = 1 + e loses the low bits of a small e; c = e - (w - 1), an exact
// difference, gives them back (c / w would be right, and is the same to one more rounding).  The rounding of |v| log2 e is
// left in: it is worth at most |v| 2^-24 of e, 2 to 3e-7 of a step size of 0.001, and giving it back costs a third of the
// function again.  -inf gives an exact zero.
__device__ __forceinline__ float softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(v) * LOG2E), w = 1.0f + e;
    return fmaxf(v, 0.f) + fmaf(__builtin_amdgcn_logf(w), 0.6931471805599453f, e - (w - 1.0f));
}

// which chunk, sample, group and channels a block has
struct ScanPlace {
    int b, g, cb, chunk, lane, wave;
    __device__ __forceinline__ ScanPlace(const Scan& a, uint32_t block, int chunks, int first) {
        const uint32_t per = (uint32_t)(a.G * a.cb);
        uint32_t i = block;
        const uint32_t gc = i % per;
        i /= per;
        chunk = (int)(i % (uint32_t)chunks) + first;
        b = (int)(i / (uint32_t)chunks);
        g = (int)gc / a.cb;
        cb = (int)gc % a.cb;
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    }
};

// A block's 64 rows of a tensor at a tile: one address for the whole block, and offsets of 32 bits to a thread's channel and
// tokens (64 L values reach 2^32 bytes at 2^24 tokens, the longest row taken).  left: tokens from the tile's start to the
// row's end; whether all 16 are there is the same for the whole block.
struct ScanTile {
    int64_t at; int left;
    __device__ __forceinline__ bool full() const { return left >= ST; }
};

// four tokens of one channel
template <typename T> struct Quad {
    Raw<T, 4> r;
    __device__ __forceinline__ void load(const void* tensor, const ScanTile& tl, uint32_t row, int q) {
        const char* p = reinterpret_cast<const char*>(static_cast<const T*>(tensor) + tl.at);
        if (tl.full()) { r.load(reinterpret_cast<const T*>(p + (row + q * 4) * (uint32_t)sizeof(T))); return; }
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = q * 4 + i < tl.left ? q * 4 + i : tl.left - 1;
            const float w = Store<T>::get(*reinterpret_cast<const T*>(p + (row + t) * (uint32_t)sizeof(T)));
            v[i] = q * 4 + i < tl.left ? w : 0.f;
        }
        r.pack(v);
    }
    static __device__ __forceinline__ void put(void* tensor, const ScanTile& tl, uint32_t row, int q, bool ok, const float (&v)[4]) {
        if (!ok) return;
        char* p = reinterpret_cast<char*>(static_cast<T*>(tensor) + tl.at);
        if (tl.full()) {
            Raw<T, 4> o;
            o.pack(v);
            o.store(reinterpret_cast<T*>(p + (row + q * 4) * (uint32_t)sizeof(T)));
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (q * 4 + i < tl.left) *reinterpret_cast<T*>(p + (row + q * 4 + i) * (uint32_t)sizeof(T)) = Store<T>::put(v[i]);
    }
};

// The rank-one updates of a wave's 64 channels x 4 states, state += (a token's B or C) x (a value a channel), are one matrix
// instruction instead of four multiply-adds: v_mfma_f32_4x4x1 with 16 blocks of 4 states x 4 channels, whose result lies as
// the states do (lane = channel, register = state).  Its first operand is broadcast from one block of four lanes, so ONE
// register holds the 16 tokens x 4 states of a tile (lane 4 t + s: token t, state s).
typedef float f32x4v __attribute__((ext_vector_type(4)));
template <int TOKEN> __device__ __forceinline__ void rank_one(float tile, float value, float (&h)[4]) {
    const f32x4v c = {h[0], h[1], h[2], h[3]};
    const f32x4v r = __builtin_amdgcn_mfma_f32_4x4x1f32(tile, value, c, 4, TOKEN, 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) h[s] = r[s];
}
// A wave's share of B or C at a tile in that form: token lane / 4, state 4 wave + lane % 4, zero behind the last state or token.
// The loads touch four rows of 16 tokens.  (31 rows of 2^24 values are the furthest offset: below 2^31 bytes.)
template <typename T> struct TileOperand {
    const T* base; uint32_t row; int t; bool in;
    __device__ __forceinline__ TileOperand(const void* m, const Scan& a, int64_t bg, int wave, int lane) {
        const int n = wave * 4 + (lane & 3);
        in = n < a.N;
        base = static_cast<const T*>(m) + bg * a.N * a.L;
        row = in ? (uint32_t)n * (uint32_t)a.L : 0u;
        t = lane >> 2;
    }
    __device__ __forceinline__ float load(int tile, int left) const {
        const char* p = reinterpret_cast<const char*>(base + (int64_t)tile * ST);
        const float v = Store<T>::get(*reinterpret_cast<const T*>(p + (row + (t < left ? t : left - 1)) * (uint32_t)sizeof(T)));
        return in && t < left ? v : 0.f;
    }
};
// Where a state's B or C multiplies a sum of its own instead, the wave reads the four of a token back from LDS, one
// 16-byte read at the same address for all lanes.  (As scalar loads from a copy laid out for it they came back in any order: a
// wait for one was a wait for all and for the LDS reads between, and the copy was a launch of its own.)
// The four stand in the padding of the token's row of the wave's shares: 1 KiB more of LDS would cost the forward kernel a
// block a compute unit (262 -> 302 us).
struct Four { float v[4]; };
__device__ __forceinline__ void keep_fours(float (&rows)[ST][SROW], int lane, float operand) { rows[lane >> 2][SC + (lane & 3)] = operand; }
__device__ __forceinline__ Four four_at(const float (&rows)[ST][SROW], int token) {
    const f32x4v q = *reinterpret_cast<const f32x4v*>(&rows[token][SC]);
    return {{q[0], q[1], q[2], q[3]}};
}
// f(0), f(1), .. as constants (the token of a matrix instruction is part of it)
template <int... I, typename F> __device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void each(F&& f) { each_of(std::make_integer_sequence<int, N>{}, f); }

// a block of W waves has 64 channels x 4 quads of a tile to load: items per thread
template <int W> struct ScanItems { static constexpr int N = W >= 4 ? 1 : 4 / W; };

// the channel, quad and row of one of a thread's items; a thread without one reads channel 0 and writes nothing
template <int W> struct ScanItem {
    int r, q, d; bool ok; uint32_t row;
    __device__ __forceinline__ ScanItem() {}
    __device__ __forceinline__ void set(const Scan& a, const ScanPlace& p, int k) {
        const int i = threadIdx.x + k * 64 * W;
        r = (i >> 2) & 63;
        q = i & 3;
        d = p.g * a.Dg + p.cb * SC + r;
        ok = i < 256 && p.cb * SC + r < a.Dg;
        row = ok ? (uint32_t)r * (uint32_t)a.L : 0u;
    }
    static __device__ __forceinline__ bool has(int k) { return W <= 4 || threadIdx.x < 256; }
};
__device__ __forceinline__ ScanTile scan_tile(const Scan& a, const ScanPlace& p, int tile) {
    const int64_t t = (int64_t)tile * ST;
    return {((int64_t)p.b * a.D + p.g * a.Dg + p.cb * SC) * a.L + t, (int)(a.L - t < ST ? a.L - t : ST)};
}

__device__ __forceinline__ float step_size(const Scan& a, float raw) { return a.softplus ? softplus(raw) : raw; }

// A rate is at most 2^100: an infinite one (a state without memory) times a step size of zero is no number, and such a token, in
// padding or behind the row's end in a tile, has to leave the state alone, and to have a gradient of zero (the rate times a
// state and its gradient must not overflow).  2^100 times any step size above 1e-28 decays as infinity does.
__device__ __forceinline__ float finite_rate(float A) {
    return fabsf(A) > 0x1p100f ? copysignf(0x1p100f, A) : A;               // (what is no number stays so)
}
// A of the lane's channel and four states; zero where there are none, so that they stay zero
__device__ __forceinline__ void load_rates(const Scan& a, int d, bool ok, int wave, float (&A)[4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) A[s] = ok && wave * 4 + s < a.N ? finite_rate(a.A[(int64_t)d * a.N + wave * 4 + s]) : 0.f;
}

// dt of four tokens: zero where there is no channel (all: the block has 64) or token, so that nothing there moves a state
template <typename T>
__device__ __forceinline__ void step_sizes(const Scan& a, const Quad<T>& qd, float bias, const ScanTile& tl, int q, bool ok,
                                           bool all, float (&raw)[4], float (&dt)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        raw[i] = qd.r.get(i) + bias;
        dt[i] = step_size(a, raw[i]);
    }
    if (!all || !tl.full()) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!ok || q * 4 + i >= tl.left) dt[i] = 0.f;
    }
}
template <typename T>
__device__ __forceinline__ float gate_of(const Quad<T>& z, int i) {
    const float v = z.r.get(i);
    return v * sigmoid(v);
}

// ---- what a chunk adds to the state behind it (REV: to the state's gradient before it), and the sum of its dt -------
// 8 x 384 x 16384 bf16 of 16 states: 163 us, REV with a gate 180 (4.9 and 4.5 T state updates a second).  Its 18.5 and 20.5 vector
// instructions a token and wave, softplus (and gate) among them, come to 98 and 108 us at the bare rates of eight waves; a wave issues 27 % of its
// time, waits 46 % for its turn and 27 % at counters and the two barriers of a tile.
template <typename T, int W, bool Z, bool REV>
__global__ void __launch_bounds__(64 * W, 8)                               // (eight waves a SIMD: at most 64 registers, and the matrix results stay in them)
scan_chunk_kernel(const Scan a) {
    constexpr int NI = ScanItems<W>::N;
    __shared__ float dts[ST][SROW], us[ST][SROW];
    const ScanPlace p(a, block_index<64 * W>(), a.nchunk - 1, REV ? 1 : 0);
    if (p.b >= a.B) return;
    const int d = p.g * a.Dg + p.cb * SC + p.lane;
    const bool ok = p.cb * SC + p.lane < a.Dg;
    const bool whole = p.cb * SC + SC <= a.Dg;
    float A[4], h[4] = {0.f, 0.f, 0.f, 0.f}, sum[NI];                       // sum: of the dt of the thread's own tokens
    load_rates(a, d, ok, p.wave, A);
#pragma unroll
    for (int s = 0; s < 4; ++s) A[s] *= LOG2E;
    const int t0 = p.chunk * a.per_chunk, t1 = t0 + a.per_chunk < a.tiles ? t0 + a.per_chunk : a.tiles;
    const TileOperand<T> op(REV ? a.Cm : a.Bm, a, (int64_t)p.b * a.G + p.g, p.wave, p.lane);
    ScanItem<W> it[NI];
    float bias[NI], vbn;
    Quad<T> qd[NI], qx[NI], qz[NI];
    auto fetch = [&](int tile) {
        const ScanTile tl = scan_tile(a, p, tile);
        vbn = op.load(tile, tl.left);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            qd[k].load(a.delta, tl, it[k].row, it[k].q);
            qx[k].load(REV ? a.dy : a.x, tl, it[k].row, it[k].q);
            if constexpr (REV && Z) qz[k].load(a.z, tl, it[k].row, it[k].q);
        }
    };
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        it[k].set(a, p, k);
        bias[k] = a.dbias && it[k].ok ? a.dbias[it[k].d] : 0.f;
        sum[k] = 0.f;
    }
    fetch(REV ? t1 - 1 : t0);
    for (int n = 0; n < t1 - t0; ++n) {
        const int tile = REV ? t1 - 1 - n : t0 + n;
        const ScanTile tl = scan_tile(a, p, tile);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            float raw[4], dt[4];
            step_sizes<T>(a, qd[k], bias[k], tl, it[k].q, it[k].ok, whole, raw, dt);
            sum[k] += (dt[0] + dt[1]) + (dt[2] + dt[3]);
            if (ScanItem<W>::has(k)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float u = qx[k].r.get(i);
                    if constexpr (REV) {
                        if constexpr (Z) u *= gate_of(qz[k], i);
                        if (!whole && !it[k].ok) u = 0.f;
                    } else u *= dt[i];
                    dts[it[k].q * 4 + i][it[k].r] = dt[i];
                    us[it[k].q * 4 + i][it[k].r] = u;
                }
            }
        }
        const float vb = vbn;
        if (n + 1 < t1 - t0) fetch(REV ? tile - 1 : tile + 1);
        __syncthreads();
        each<ST>([&](auto I) {
            constexpr int i = REV ? ST - 1 - I : I;
            const float dt = dts[i][p.lane], u = us[i][p.lane];
            float decay[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) decay[s] = __builtin_amdgcn_exp2f(dt * A[s]);
            if constexpr (REV) rank_one<i>(vb, u, h);
#pragma unroll
            for (int s = 0; s < 4; ++s) h[s] *= decay[s];
            if constexpr (!REV) rank_one<i>(vb, u, h);
        });
        __syncthreads();
    }
    const int64_t c = (int64_t)p.b * a.nchunk + p.chunk;
    if (ok) {
#pragma unroll
        for (int s = 0; s < 4; ++s) a.cst[(c * 4 * W + p.wave * 4 + s) * a.D + d] = h[s];
    }
#pragma unroll
    for (int k = 0; k < NI; ++k) {
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) sum[k] += __shfl_xor(sum[k], off, 64);
        if (it[k].ok && it[k].q == 0) a.cdt[c * a.D + it[k].d] = sum[k];
    }
}

// ---- the chunks' own states, one behind the other: cst[c] becomes the state that chunk c starts from (REV: the
// state's gradient behind it).  A block has 64 channels and one state; its waves take a run of chunks each, side by side,
// chain the runs through LDS and walk their run again: four waves with up to 8 chunks each, or 16 with 16; what a run of that
// length reads stays in registers for the second walk: 5.7 us for 32 chunks of 8 x 384 channels, 8.4 for 256 of 192.  (Chained in front of every chunk by the scan's own blocks, the
// states are read as often as there are chunks: 503 MB from the caches for 256 chunks of 192 channels, 45 us instead of 20.)
// A chunk's decay leaves the range of fp32 where the states on both sides of it need not (1e30 times e^-100, or a growing state,
// A > 0, of 1e-30 times e^100): it is applied as its square root, twice.  A state of zero stays zero over any growth: 0 times
// infinity is no number.
__device__ __forceinline__ float over_chunk(float h, float sum, float A, float own) {
    const float root = __builtin_amdgcn_exp2f(0.5f * sum * A);
    return h == 0.f ? own : fmaf(root * h, root, own);
}
template <bool REV, int RUNS, int LEN>
__global__ void __launch_bounds__(64 * RUNS)
scan_chain_kernel(const Scan a, int states) {
    __shared__ float sums[RUNS][64], own[RUNS][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int d = blockIdx.x * 64 + lane, n = blockIdx.y, b = blockIdx.z;
    const bool ok = d < a.D;
    const int dr = ok ? d : 0;
    const float A = n < a.N ? finite_rate(a.A[(int64_t)dr * a.N + n]) * LOG2E : 0.f;
    const int per = (a.nchunk + RUNS - 1) / RUNS, c0 = run * per, c1 = c0 + per < a.nchunk ? c0 + per : a.nchunk;
    float* st = a.cst + ((int64_t)b * a.nchunk * states + n) * a.D;        // chunk c: + c states D
    const float* dt = a.cdt + (int64_t)b * a.nchunk * a.D;
    // chunk c on the way; the last one has nothing behind it and left no state
    auto read = [&](int c, float& t, float& v) {
        const bool in = c < c1 && c < a.nchunk - 1;
        const int64_t k = REV ? a.nchunk - 1 - (in ? c : 0) : (in ? c : 0);
        t = dt[k * a.D + dr];
        v = st[k * states * a.D + dr];
        if (!in) { t = 0.f; v = 0.f; }
    };
    float sum = 0.f, h = 0.f, t[LEN], v[LEN];
    for (int c = c0; c < c1; c += LEN) {
#pragma unroll
        for (int j = 0; j < LEN; ++j) read(c + j, t[j], v[j]);
#pragma unroll
        for (int j = 0; j < LEN; ++j) {
            sum += t[j];
            h = over_chunk(h, t[j], A, v[j]);
        }
    }
    sums[run][lane] = sum;
    own[run][lane] = h;
    __syncthreads();
    const float* first = REV ? a.dlast : a.h0;
    h = first && n < a.N ? first[((int64_t)b * a.D + dr) * a.N + n] : 0.f;
    for (int r = 0; r < run; ++r) h = over_chunk(h, sums[r][lane], A, own[r][lane]);
    for (int c = c0; c < c1; c += LEN) {
        if (c1 - c0 > LEN) {
#pragma unroll
            for (int j = 0; j < LEN; ++j) read(c + j, t[j], v[j]);
        }
#pragma unroll
        for (int j = 0; j < LEN; ++j)
            if (c + j < c1) {
                const int64_t k = REV ? a.nchunk - 1 - (c + j) : c + j;
                if (ok) st[k * states * a.D + d] = h;
                h = over_chunk(h, t[j], A, v[j]);
            }
    }
}
// what a block starts from: the chained state of its chunk, or the call's own
template <int W>
__device__ __forceinline__ float start_state(const Scan& a, const ScanPlace& p, int d, bool ok, int s, const float* first) {
    if (!ok) return 0.f;
    if (a.nchunk > 1) return (a.cst + (((int64_t)p.b * a.nchunk + p.chunk) * 4 * W + p.wave * 4 + s) * a.D)[(uint32_t)d];
    return first && p.wave * 4 + s < a.N ? first[((int64_t)p.b * a.D + d) * a.N + p.wave * 4 + s] : 0.f;
}

// ---- forward ------------------------------------------------------------------------------------------------------
// 8 x 384 x 16384 bf16 of 16 states, gated, the states before every tile kept: 257 us (3.1 T state updates a second; 604 MB, 2.3
// TB/s).  At most 80 registers and, with 16 states, 25.5 KiB: six blocks a compute unit.  Its 28 vector instructions a token and
// wave, five of them exponentials and the like, come to 138 us at the bare rates of eight waves; a wave issues 24 % of its
// time, waits 42 % for its turn and 37 % at LDS, counters and barriers.
template <typename T, int W, bool Z>
__global__ void __launch_bounds__(64 * W, 6)
scan_fwd_kernel(const Scan a) {
    constexpr int NI = ScanItems<W>::N;
    __shared__ __attribute__((aligned(16))) float dts[ST][SROW], us[ST][SROW], part[W][ST][SROW];
    const ScanPlace p(a, block_index<64 * W>(), a.nchunk, 0);
    if (p.b >= a.B) return;
    const int d = p.g * a.Dg + p.cb * SC + p.lane;
    const bool ok = p.cb * SC + p.lane < a.Dg, whole = p.cb * SC + SC <= a.Dg;
    const int64_t bg = (int64_t)p.b * a.G + p.g;
    const TileOperand<T> opb(a.Bm, a, bg, p.wave, p.lane), opc(a.Cm, a, bg, p.wave, p.lane);
    const int t0 = p.chunk * a.per_chunk, t1 = t0 + a.per_chunk < a.tiles ? t0 + a.per_chunk : a.tiles;
    ScanItem<W> it[NI];
    float bias[NI], skip[NI], vbn, vcn;
    Quad<T> qd[NI], qx[NI], qz[NI];
    auto fetch = [&](int tile) {
        const ScanTile tl = scan_tile(a, p, tile);
        vbn = opb.load(tile, tl.left);
        vcn = opc.load(tile, tl.left);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            qd[k].load(a.delta, tl, it[k].row, it[k].q);
            qx[k].load(a.x, tl, it[k].row, it[k].q);
            if constexpr (Z) qz[k].load(a.z, tl, it[k].row, it[k].q);
        }
    };
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        it[k].set(a, p, k);
        bias[k] = a.dbias && it[k].ok ? a.dbias[it[k].d] : 0.f;
        skip[k] = a.Dskip && it[k].ok ? a.Dskip[it[k].d] : 0.f;
    }
    fetch(t0);
    float A[4], h[4];
    load_rates(a, d, ok, p.wave, A);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        A[s] *= LOG2E;
        h[s] = start_state<W>(a, p, d, ok, s, a.h0);
    }
    for (int tile = t0; tile < t1; ++tile) {
        const float vb = vbn;
        const ScanTile tl = scan_tile(a, p, tile);
        float x[NI][4], gate[NI][4];
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            float raw[4], dt[4];
            step_sizes<T>(a, qd[k], bias[k], tl, it[k].q, it[k].ok, whole, raw, dt);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[k][i] = qx[k].r.get(i);
                if constexpr (Z) gate[k][i] = gate_of(qz[k], i);
                if (ScanItem<W>::has(k)) {
                    dts[it[k].q * 4 + i][it[k].r] = dt[i];
                    us[it[k].q * 4 + i][it[k].r] = dt[i] * x[k][i];
                }
            }
        }
        keep_fours(part[p.wave], p.lane, vcn);
        if (tile + 1 < t1) fetch(tile + 1);
        __syncthreads();
        if (a.ckpt && ok) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
                (a.ckpt + (((int64_t)p.b * a.tiles + tile) * 4 * W + p.wave * 4 + s) * a.D)[(uint32_t)d] = h[s];
        }
        each<ST>([&](auto I) {
            constexpr int i = I;
            const float dt = dts[i][p.lane], u = us[i][p.lane];
            const Four cv = four_at(part[p.wave], i);
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) h[s] *= __builtin_amdgcn_exp2f(dt * A[s]);
            rank_one<i>(vb, u, h);
#pragma unroll
            for (int s = 0; s < 4; ++s) y = fmaf(cv.v[s], h[s], y);
            part[p.wave][i][p.lane] = y;
        });
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            if (!ScanItem<W>::has(k)) continue;
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[i] = skip[k] * x[k][i];
#pragma unroll
                for (int w = 0; w < W; ++w) y[i] += part[w][it[k].q * 4 + i][it[k].r];
                if constexpr (Z) y[i] *= gate[k][i];
            }
            Quad<T>::put(a.y, tl, it[k].row, it[k].q, it[k].ok, y);
        }
    }
    if (a.last && ok && t1 == a.tiles) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (p.wave * 4 + s < a.N) a.last[((int64_t)p.b * a.D + d) * a.N + p.wave * 4 + s] = h[s];
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------
// Sums over the 64 lanes, many values at a time: where a butterfly would add a value to itself in both halves, two
// values swap halves first, so that every step halves the number of values (8 values of 8 tokens: 141 instructions
// instead of 384 for 64 butterflies).
__device__ __forceinline__ float halves32(float a, float b) {              // lanes 0-31: a's sum, 32-63: b's
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float halves16(float a, float b) {              // even rows of 16 lanes: a's, odd rows: b's
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// lanes with `hi` unset: a's sum with the lane that CTRL names, with it set: b's
template <int CTRL> __device__ __forceinline__ float halves_dpp(float a, float b, bool hi) {
    return (hi ? b : a) + dpp<CTRL>(hi ? a : b);
}
constexpr int DPP_ROR8 = 0x128, DPP_HALF_MIRROR = 0x141, DPP_XOR2 = 0x4E, DPP_XOR1 = 0xB1;
// the shares of dB (v[0..3]) and dC (v[4..7]) of one token: lane l holds value 4 (l >> 5) + 2 (l >> 4 & 1) + (l >> 3 & 1),
// still to be added over its group of eight lanes
__device__ __forceinline__ float lanes_fold(const float (&v)[8], int lane) {
    float h[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) h[s] = halves32(v[s], v[4 + s]);
    return halves_dpp<DPP_ROR8>(halves16(h[0], h[2]), halves16(h[1], h[3]), lane & 8);
}
// those of eight tokens: lane l holds the finished value of token l & 7
__device__ __forceinline__ float tokens_fold(const float (&w)[8], int lane) {
    float q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = halves_dpp<DPP_HALF_MIRROR>(w[k], w[k + 4], lane & 4);
    return halves_dpp<DPP_XOR1>(halves_dpp<DPP_XOR2>(q[0], q[2], lane & 2), halves_dpp<DPP_XOR2>(q[1], q[3], lane & 2), lane & 1);
}

// WHOLE: the block has 64 channels.  Where it has fewer, the shares of the lanes without one are taken out: they are
// zero only as long as B and C are finite.
template <typename T, int W, bool Z, bool WHOLE>
__device__ __forceinline__ void scan_bwd_body(const Scan& a, const ScanPlace& p, float* smem) {
    constexpr int NI = ScanItems<W>::N;
    float (*dts)[SROW] = reinterpret_cast<float (*)[SROW]>(smem);
    float (*us)[SROW] = dts + ST;
    float (*es)[SROW] = us + ST;
    float (*part0)[ST][SROW] = reinterpret_cast<float (*)[ST][SROW]>(es + ST);          // [W]: shares of sum g B
    float (*part1)[ST][SROW] = part0 + W;                                               // [W]: shares of sum A a g h
    float (*part2)[ST][SROW] = part1 + W;                                               // [W], with z: shares of s
    const int d = p.g * a.Dg + p.cb * SC + p.lane;
    const bool ok = WHOLE || p.cb * SC + p.lane < a.Dg;
    const int dr = ok ? d : 0;
    const int t0 = p.chunk * a.per_chunk, t1 = t0 + a.per_chunk < a.tiles ? t0 + a.per_chunk : a.tiles;
    ScanItem<W> it[NI];
    float bias[NI], skip[NI], dD[NI], db[NI];
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        it[k].set(a, p, k);
        bias[k] = a.dbias && it[k].ok ? a.dbias[it[k].d] : 0.f;
        skip[k] = a.Dskip && it[k].ok ? a.Dskip[it[k].d] : 0.f;
        dD[k] = 0.f;
        db[k] = 0.f;
    }
    Quad<T> qd[NI], qx[NI], qy[NI], qz[NI];
    float hn[4], vbn, vcn;
    const int64_t bg = (int64_t)p.b * a.G + p.g;
    const TileOperand<T> opb(a.Bm, a, bg, p.wave, p.lane), opc(a.Cm, a, bg, p.wave, p.lane);
    auto fetch = [&](int tile) {
        const ScanTile tl = scan_tile(a, p, tile);
        vbn = opb.load(tile, tl.left);
        vcn = opc.load(tile, tl.left);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            qd[k].load(a.delta, tl, it[k].row, it[k].q);
            qx[k].load(a.x, tl, it[k].row, it[k].q);
            qy[k].load(a.dy, tl, it[k].row, it[k].q);
            if constexpr (Z) qz[k].load(a.z, tl, it[k].row, it[k].q);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) hn[s] = (a.ckpt + (((int64_t)p.b * a.tiles + tile) * 4 * W + p.wave * 4 + s) * a.D)[(uint32_t)dr];
    };
    fetch(t1 - 1);
    float A[4], A2[4], g[4], dA[4] = {0.f, 0.f, 0.f, 0.f};
    load_rates(a, d, ok, p.wave, A);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        A2[s] = A[s] * LOG2E;
        g[s] = start_state<W>(a, p, d, ok, s, a.dlast);
    }
    float* bco = a.bcpart + (((int64_t)p.cb * a.B * a.G + bg) * a.tiles * 2 * W + p.wave) * 64;
    for (int tile = t1 - 1; tile >= t0; --tile) {
        const ScanTile tl = scan_tile(a, p, tile);
        float x[NI][4], raw[NI][4], slope[NI][4];                               // slope: dy silu'(z)
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            float dt[4];
            step_sizes<T>(a, qd[k], bias[k], tl, it[k].q, it[k].ok, WHOLE, raw[k], dt);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[k][i] = qx[k].r.get(i);
                float e = WHOLE || it[k].ok ? qy[k].r.get(i) : 0.f;
                if constexpr (Z) {
                    const float z = qz[k].r.get(i), q = sigmoid(z);
                    slope[k][i] = e * (q * fmaf(z, 1.0f - q, 1.0f));
                    e *= z * q;
                }
                if (ScanItem<W>::has(k)) {
                    dts[it[k].q * 4 + i][it[k].r] = dt[i];
                    us[it[k].q * 4 + i][it[k].r] = dt[i] * x[k][i];
                    es[it[k].q * 4 + i][it[k].r] = e;
                }
            }
        }
        float hs[ST + 1][4], as[ST][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) hs[0][s] = ok ? hn[s] : 0.f;
        const float vb = vbn, vc = vcn;
        keep_fours(part0[p.wave], p.lane, vb);
        if constexpr (Z) keep_fours(part1[p.wave], p.lane, vc);
        __syncthreads();
        // the operands of the next token are read while one is worked on: two waves a SIMD do not hide the reads
        float dt, u, e, dtn, un, en;
        Four m, mn;
        auto ask = [&](int i, bool back) {
            dtn = dts[i][p.lane];
            un = us[i][p.lane];
            if (back) { en = es[i][p.lane]; mn = four_at(part0[p.wave], i); }
            else if constexpr (Z) mn = four_at(part1[p.wave], i);
        };
        auto take = [&]() { dt = dtn; u = un; e = en; m = mn; };
        ask(0, false);
        each<ST>([&](auto I) {
            constexpr int i = I;
            take();
            ask(i + 1 < ST ? i + 1 : ST - 1, i + 1 == ST);
            __builtin_amdgcn_sched_barrier(0);
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                as[i][s] = __builtin_amdgcn_exp2f(dt * A2[s]);
                hs[i + 1][s] = as[i][s] * hs[i][s];
            }
            rank_one<i>(vb, u, hs[i + 1]);
            if constexpr (Z) {
#pragma unroll
                for (int s = 0; s < 4; ++s) y = fmaf(m.v[s], hs[i + 1][s], y);
                part2[p.wave][i][p.lane] = y;
            }
        });
        float tA[4] = {0.f, 0.f, 0.f, 0.f}, fold[8];
        each<ST>([&](auto I) {
            constexpr int i = ST - 1 - I;
            take();
            if constexpr (i > 0) ask(i - 1, true);
            if (i == ST / 2 && tile > t0) fetch(tile - 1);                 // (half of the states are done with: registers are free)
            __builtin_amdgcn_sched_barrier(0);
            float gB = 0.f, gA = 0.f, pr[8];
            rank_one<i>(vc, e, g);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                pr[s] = g[s] * u;
                pr[4 + s] = hs[i + 1][s] * e;
                gB = fmaf(g[s], m.v[s], gB);
                g[s] *= as[i][s];
                const float q = g[s] * hs[i][s];
                gA = fmaf(A[s], q, gA);
                tA[s] = fmaf(dt, q, tA[s]);
            }
            part0[p.wave][i][p.lane] = gB;
            part1[p.wave][i][p.lane] = gA;
            if constexpr (!WHOLE) {
#pragma unroll
                for (int s = 0; s < 8; ++s) pr[s] = ok ? pr[s] : 0.f;
            }
            fold[i & 7] = lanes_fold(pr, p.lane);
            if ((i & 7) == 0) (bco + ((int64_t)tile * 2 + (i >> 3)) * W * 64)[(uint32_t)p.lane] = tokens_fold(fold, p.lane);
        });
#pragma unroll
        for (int s = 0; s < 4; ++s) dA[s] += tA[s];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            if (!ScanItem<W>::has(k)) continue;
            float ox[4], od[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float gB = 0.f, gA = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    gB += part0[w][it[k].q * 4 + i][it[k].r];
                    gA += part1[w][it[k].q * 4 + i][it[k].r];
                }
                const float dti = dts[it[k].q * 4 + i][it[k].r], ei = es[it[k].q * 4 + i][it[k].r];
                ox[i] = fmaf(gB, dti, skip[k] * ei);
                od[i] = fmaf(gB, x[k][i], gA);
                if (a.softplus) od[i] *= sigmoid(raw[k][i]);
                dD[k] = fmaf(ei, x[k][i], dD[k]);
                if (it[k].q * 4 + i < tl.left) db[k] += od[i];              // (behind the row g is the last state's gradient)
            }
            Quad<T>::put(a.dx, tl, it[k].row, it[k].q, it[k].ok, ox);
            Quad<T>::put(a.ddelta, tl, it[k].row, it[k].q, it[k].ok, od);
            if constexpr (Z) {
                float oz[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float y = skip[k] * x[k][i];
#pragma unroll
                    for (int w = 0; w < W; ++w) y += part2[w][it[k].q * 4 + i][it[k].r];
                    oz[i] = slope[k][i] * y;
                }
                Quad<T>::put(a.dz, tl, it[k].row, it[k].q, it[k].ok, oz);
            }
        }
        // (no barrier: what the next tile's first part overwrites are the thread's own tokens, and the shares are not
        // written before the barrier behind it)
    }
    const int64_t c = (int64_t)p.b * a.nchunk + p.chunk;
    if (ok) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            a.dApart[(c * 4 * W + p.wave * 4 + s) * a.D + d] = dA[s];
            if (a.dh0 && p.chunk == 0 && p.wave * 4 + s < a.N) a.dh0[((int64_t)p.b * a.D + d) * a.N + p.wave * 4 + s] = g[s];
        }
    }
#pragma unroll
    for (int k = 0; k < NI; ++k) {
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
            dD[k] += __shfl_xor(dD[k], off, 64);
            db[k] += __shfl_xor(db[k], off, 64);
        }
        if (it[k].ok && it[k].q == 0) {
            a.dDpart[(c * 2 + 0) * a.D + it[k].d] = dD[k];
            a.dDpart[(c * 2 + 1) * a.D + it[k].d] = db[k];
        }
    }
}

// 8 x 384 x 16384 bf16 of 16 states, gated: 782 us (1.0 T state updates a second): the 256 registers that hold the tile's states and
// decays leave two waves a SIMD.  85 vector instructions a token and wave come to 435 us at the bare rates of two waves; a
// wave issues 47 % of its time, waits 16 % for its turn and 37 % at LDS, counters and barriers, which one other wave does not cover.
// Both bodies in one kernel spill 32 registers with a gate and 16 states, nearly all before the loop.
template <typename T, int W, bool Z>
__global__ void __launch_bounds__(64 * W, W >= 4 ? 2 : 1)                  // (fewer waves have more tokens a lane: 256 registers would spill)
scan_bwd_kernel(const Scan a) {
    extern __shared__ __attribute__((aligned(16))) float smem[];
    const ScanPlace p(a, block_index<64 * W>(), a.nchunk, 0);
    if (p.b >= a.B) return;
    if (p.cb * SC + SC <= a.Dg) scan_bwd_body<T, W, Z, true>(a, p, smem);
    else scan_bwd_body<T, W, Z, false>(a, p, smem);
}

// What the backward kernel's blocks left in shares, each sum in a fixed order: the first `bcs` blocks take dB and dC
// [B][G][N][L] from the channel blocks' shares (a thread has one token and a state of four, so writes are whole lines), the
// others dA [D][N], dD and dbias [D] from those of all samples and chunks (rows 0 .. N-1 are dA's states, N is dD, N + 1
// dbias; lanes run along the channels).
template <typename T>
__global__ void __launch_bounds__(256)
scan_reduce_kernel(const Scan a, int W, int bcs, float* __restrict__ dA, float* __restrict__ dD, float* __restrict__ dbias) {
    const uint32_t block = block_index<256>();
    if (block < (uint32_t)bcs) {
        const int across = (int)((a.L + 63) / 64);
        const int64_t t = (int64_t)(block % across) * 64 + (threadIdx.x & 63);
        const int64_t bg = block / across, groups = (int64_t)a.tiles * 2, stride = (int64_t)a.B * a.G * groups * W * 64;
        if (t >= a.L) return;
        T *dB = static_cast<T*>(a.dB), *dC = static_cast<T*>(a.dC);
        for (int n = threadIdx.x >> 6; n < a.N; n += 4) {
            const float* p = a.bcpart + ((bg * groups + (t >> 3)) * W + (n >> 2)) * 64 + ((n >> 1) & 1) * 16 + (n & 1) * 8 + (t & 7);
            float b = 0.f, c = 0.f;
            for (int k = 0; k < a.cb; ++k) {
                b += p[k * stride];
                c += p[k * stride + 32];
            }
            dB[(bg * a.N + n) * a.L + t] = Store<T>::put(b);
            dC[(bg * a.N + n) * a.L + t] = Store<T>::put(c);
        }
        return;
    }
    __shared__ float red[16][17];
    const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, wide = (a.D + 15) / 16;
    const int i = (int)(block - bcs), d = i % wide * 16 + col, row = i / wide, n = a.B * a.nchunk;
    float s = 0.f;
    if (row > a.N + 1) return;
    if (d < a.D) {
        const float* p = row < a.N ? a.dApart + (int64_t)row * a.D + d : a.dDpart + (int64_t)(row - a.N) * a.D + d;
        const int64_t step = (int64_t)(row < a.N ? 4 * W : 2) * a.D;
#pragma unroll 8
        for (int c = slice; c < n; c += 16) s += p[c * step];
    }
    red[slice][col] = s;
    __syncthreads();
    for (int h = 8; h > 0; h >>= 1) {
        if (slice < h) red[slice][col] += red[slice + h][col];
        __syncthreads();
    }
    if (slice != 0 || d >= a.D) return;
    if (row < a.N) dA[(int64_t)d * a.N + row] = red[0][col];
    else if (row == a.N) { if (dD) dD[d] = red[0][col]; }
    else if (dbias) dbias[d] = red[0][col];
}

// ---- one token -----------------------------------------------------------------------------------------------------
// NL lanes share a channel, four states each.  Bound by the state's 8 N bytes per channel (256 x 768 of 16 states: 9.7 us, 2.6
// TB/s; 1 x 384: 3.5 us, a launch).  state_out may be the state.
template <typename T, int NL>
__global__ void __launch_bounds__(256)
scan_update_kernel(const T* __restrict__ x, const T* __restrict__ delta, const float* __restrict__ A, const T* __restrict__ Bm,
                   const T* __restrict__ Cm, const float* __restrict__ Dskip, const T* __restrict__ z,
                   const float* __restrict__ dbias, const float* state, float* state_out, T* __restrict__ y, int64_t n, int D, int G,
                   int N, int soft) {
    const int64_t i = (int64_t)block_index<256>() * (256 / NL) + threadIdx.x / NL;
    const int lane = threadIdx.x % NL;
    const bool live = i < n;
    float s = 0.f, xv = 0.f;
    if (live) {
        const int d = (int)((uint32_t)i % (uint32_t)D), b = (int)((uint32_t)i / (uint32_t)D);
        const int64_t bg = (int64_t)b * G + d / (D / G);
        xv = Store<T>::get(x[i]);
        float dt = Store<T>::get(delta[i]) + (dbias ? dbias[d] : 0.f);
        if (soft) dt = softplus(dt);
        const float u = dt * xv;
        float h[4], Av[4];
        const int n0 = lane * 4;
        if ((N & 3) == 0 && n0 < N) {
            Raw<float, 4> hv, av;
            hv.load(state + i * N + n0);
            av.load(A + (int64_t)d * N + n0);
            hv.unpack(h);
            av.unpack(Av);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h[k] = n0 + k < N ? state[i * N + n0 + k] : 0.f;
                Av[k] = n0 + k < N ? A[(int64_t)d * N + n0 + k] : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n0 + k < N) {
                h[k] = fmaf(exp_fast(dt * finite_rate(Av[k])), h[k], u * Store<T>::get(Bm[bg * N + n0 + k]));
                s = fmaf(Store<T>::get(Cm[bg * N + n0 + k]), h[k], s);
            }
        if ((N & 3) == 0 && n0 < N) {
            Raw<float, 4> hv;
            hv.pack(h);
            hv.store(state_out + i * N + n0);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (n0 + k < N) state_out[i * N + n0 + k] = h[k];
        }
        if (lane == 0 && Dskip) s = fmaf(Dskip[d], xv, s);
    }
#pragma unroll
    for (int off = NL / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (live && lane == 0) {
        if (z) { const float zv = Store<T>::get(z[i]); s *= zv * sigmoid(zv); }
        y[i] = Store<T>::put(s);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
static int scan_waves(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8; }

// How many chunks a row is cut into.  A compute unit holds six blocks of the forward kernel or two of the backward.  k of them
// side by side do not take k times one block's share of the vector pipe: a SIMD issues 39, 73, 84 and 93 multiply-adds a
// clock and compute unit with one, two, four and eight waves, so one alone takes 2.4 shares (backward 1.9) and k take about
// k + 1/2 (backward k).  Chunks cost the pass over their own states, 0.6 of the forward kernel's time and 0.2 of the
// backward's, a block about half a tile beside its tiles, and the chain about three.  The number that costs least is
// taken, chunks of at least two tiles.  Measured, 8 x 384 x 16384 bf16 of 16 states: forward 784, 546, 463, 449, 440, 454 us with 5, 10, 16,
// 21, 32, 48 chunks, backward 1497, 1068, 1065, 1020, 1020, 1047; one 16384-token prompt of 192 channels 70, 61, 53, 46, 45, 46
// us with 64, 85, 128, 171, 256, 512.
// The figures are those of 16 states, blocks of four waves; the other forms are planned with them.  What is chosen against the best of
// eleven counts, gated bf16, us: 4 x 384 x 4096 forward 61 / 59, 64 / 59, 74 / 64, 111 / 97 with 4, 8, 16, 32 states, backward 174 / 118
// (one-wave blocks: four fit a compute unit), 147 / 145, 151 / 151, 267 / 259; 8 x 384 x 16384 forward 328 / 319, 351 / 345, 369 / 367,
// 614 / 614, backward 760 / 704, 863 / 861, 917 / 916, 1793 / 1793.
static void scan_plan(Scan* a, bool bwd) {
    a->Dg = a->D / a->G;
    a->cb = (int)cdiv(a->Dg, SC);
    a->tiles = (int)cdiv(a->L, ST);
    const int64_t blocks = (int64_t)a->B * a->G * a->cb;
    const int held = bwd ? 2 : 6;
    const double again = bwd ? 1.2 : 1.6;
    auto shares = [&](int64_t k) { return k == 0 ? 0.0 : bwd ? (k == 1 ? 1.9 : 2.0) : (k == 1 ? 2.4 : (double)k + 0.5); };
    auto cost = [&](int64_t chunks, int64_t per) {
        const int64_t k = cdiv(blocks * chunks, 256);
        return ((double)(k / held) * shares(held) + shares(k % held)) * ((double)per + 0.5);
    };
    double best = cost(1, a->tiles);
    a->per_chunk = a->tiles;
    for (int64_t k = 1; k <= 16; ++k) {                                    // k blocks a compute unit
        int64_t n = 256 * k / blocks;
        if (n > a->tiles / 2) n = a->tiles / 2;
        if (n < 2) continue;
        const int64_t per = cdiv(a->tiles, n);
        const double c = cost(cdiv(a->tiles, per), per) * again + 3.0;
        if (c < best) { best = c; a->per_chunk = (int)per; }
    }
    a->nchunk = (int)cdiv(a->tiles, a->per_chunk);
}

static int scan_check(const char* what, const rst_scan_desc* s) {
    RST_REQUIRE(s != nullptr, "%s: null descriptor", what);
    RST_REQUIRE(s->dtype == RST_DTYPE_F32 || s->dtype == RST_DTYPE_BF16, "%s: unknown dtype %d", what, s->dtype);
    RST_REQUIRE(s->B > 0 && s->D > 0 && s->L > 0, "%s: empty shape B=%d D=%d L=%lld", what, s->B, s->D, (long long)s->L);
    RST_REQUIRE(s->G > 0 && s->D % s->G == 0, "%s: D=%d not divisible by groups=%d", what, s->D, s->G);
    RST_REQUIRE(s->N > 0 && s->N <= 32, "%s: N=%d states (1 to 32)", what, s->N);
    RST_REQUIRE(s->L <= (1ll << 24) && (int64_t)s->B * s->D <= (1ll << 30) && (int64_t)s->B * s->G <= 65535,
                "%s: shape out of range B=%d D=%d G=%d L=%lld", what, s->B, s->D, s->G, (long long)s->L);
    return RST_OK;
}

static void scan_shape(Scan* a, const rst_scan_desc* s, bool bwd) {
    a->B = s->B; a->D = s->D; a->G = s->G; a->N = s->N; a->L = s->L; a->softplus = s->delta_softplus;
    scan_plan(a, bwd);
}

// Scratch of a call, carved from the caller's workspace (base == null: only measured)
static size_t scan_carve(Scan* a, char* base, bool bwd) {
    const int W = scan_waves(a->N);
    size_t off = 0;
    auto take = [&](int64_t floats) {
        float* p = base ? reinterpret_cast<float*>(base + off) : nullptr;
        off = (off + (size_t)floats * sizeof(float) + 255) & ~size_t(255);
        return p;
    };
    const int64_t chunks = (int64_t)a->B * a->nchunk;
    if (a->nchunk > 1) {
        a->cst = take(chunks * 4 * W * a->D);
        a->cdt = take(chunks * a->D);
    }
    if (bwd) {
        a->bcpart = take((int64_t)a->cb * a->B * a->G * a->tiles * 2 * W * 64);
        a->dApart = take(chunks * 4 * W * a->D);
        a->dDpart = take(chunks * 2 * a->D);
    }
    return off;
}

template <bool REV>
static int scan_chain(const Scan& a, int states, hipStream_t st) {
    const dim3 grid((unsigned)cdiv(a.D, 64), states, a.B);
    if (a.nchunk <= 32) hipLaunchKernelGGL((scan_chain_kernel<REV, 4, 8>), grid, dim3(256), 0, st, a, states);
    else hipLaunchKernelGGL((scan_chain_kernel<REV, 16, 16>), grid, dim3(1024), 0, st, a, states);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

template <typename T, int W, bool Z>
static int scan_fwd_t(const Scan& a, hipStream_t st) {
    const double n = (double)a.B * a.D * a.L;
    ProfScope prof(st, "scan_fwd", n * (7.0 * a.N + 12), sizeof(T) * n * (a.z ? 4 : 3));
    const int64_t per = (int64_t)a.B * a.G * a.cb;
    RST_REQUIRE(per * a.nchunk < (1ll << 31), "scan: grid out of range");
    if (a.nchunk > 1) {
        hipLaunchKernelGGL((scan_chunk_kernel<T, W, false, false>), grid_of<64 * W>(per * (a.nchunk - 1)), dim3(64 * W), 0, st, a);
        RST_LAUNCH_CHECK();
        RST_TRY(scan_chain<false>(a, 4 * W, st));
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, W, Z>), grid_of<64 * W>(per * a.nchunk), dim3(64 * W), 0, st, a);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

template <typename T, int W, bool Z>
static int scan_bwd_t(const Scan& a, float* dA, float* dD, float* dbias, hipStream_t st) {
    const double n = (double)a.B * a.D * a.L;
    ProfScope prof(st, "scan_bwd", n * (16.0 * a.N + 28), sizeof(T) * n * (a.z ? 7 : 5));
    const int64_t per = (int64_t)a.B * a.G * a.cb;
    RST_REQUIRE(per * a.nchunk < (1ll << 31), "scan: grid out of range");
    if (a.nchunk > 1) {
        hipLaunchKernelGGL((scan_chunk_kernel<T, W, Z, true>), grid_of<64 * W>(per * (a.nchunk - 1)), dim3(64 * W), 0, st, a);
        RST_LAUNCH_CHECK();
        RST_TRY(scan_chain<true>(a, 4 * W, st));
    }
    const size_t lds = (size_t)(3 + (Z ? 3 : 2) * W) * ST * SROW * sizeof(float);
    KernelSetup ks;
    RST_TRY(kernel_setup(reinterpret_cast<const void*>(scan_bwd_kernel<T, W, Z>), 64 * W, lds, &ks));
    hipLaunchKernelGGL((scan_bwd_kernel<T, W, Z>), grid_of<64 * W>(per * a.nchunk), dim3(64 * W), lds, st, a);
    RST_LAUNCH_CHECK();
    const int64_t bcs = cdiv(a.L, 64) * a.B * a.G, all = bcs + cdiv(a.D, 16) * (a.N + 2);
    RST_REQUIRE(all < (1ll << 31), "scan: grid out of range");
    hipLaunchKernelGGL((scan_reduce_kernel<T>), grid_of<256>(all), dim3(256), 0, st, a, W, (int)bcs, dA, dD, dbias);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

template <typename T, int NL>
static int scan_update_t(const rst_scan_desc* s, const rst_scan_inputs* in, const float* state, float* state_out, T* y, hipStream_t st) {
    const int64_t n = (int64_t)s->B * s->D;
    ProfScope prof(st, "scan_update", n * (7.0 * s->N + 20), n * 8.0 * s->N);
    hipLaunchKernelGGL((scan_update_kernel<T, NL>), grid_of<256>(cdiv(n, 256 / NL)), dim3(256), 0, st, static_cast<const T*>(in->x),
                       static_cast<const T*>(in->delta), in->A, static_cast<const T*>(in->B), static_cast<const T*>(in->C), in->D,
                       static_cast<const T*>(in->z), in->delta_bias, state, state_out, y, n, s->D, s->G, s->N, s->delta_softplus);
    RST_LAUNCH_CHECK();
    return RST_OK;
}

}  // namespace rst

using namespace rst;

#define SCAN_WAVES(CALL, T) (W == 1 ? CALL(T, 1) : W == 2 ? CALL(T, 2) : W == 4 ? CALL(T, 4) : CALL(T, 8))
#define SCAN_TYPES(CALL) (s->dtype == RST_DTYPE_F32 ? SCAN_WAVES(CALL, float) : SCAN_WAVES(CALL, bf16_t))

extern "C" {

size_t rst_scan_workspace_bytes(const rst_scan_desc* s) {
    if (scan_check("scan_workspace_bytes", s) != RST_OK) return 0;
    Scan a{};
    scan_shape(&a, s, false);
    return scan_carve(&a, nullptr, false);
}
size_t rst_scan_saved_bytes(const rst_scan_desc* s) {
    if (scan_check("scan_saved_bytes", s) != RST_OK) return 0;
    Scan a{};
    scan_shape(&a, s, true);
    return (size_t)a.B * a.tiles * 4 * scan_waves(a.N) * a.D * sizeof(float);
}
size_t rst_scan_bwd_workspace_bytes(const rst_scan_desc* s) {
    if (scan_check("scan_bwd_workspace_bytes", s) != RST_OK) return 0;
    Scan a{};
    scan_shape(&a, s, true);
    return scan_carve(&a, nullptr, true);
}

int rst_scan_fwd(const rst_scan_desc* s, const rst_scan_inputs* in, const float* state_in, void* y, float* state_out, float* saved,
                 void* workspace, size_t workspace_bytes, void* stream) {
    RST_TRY(scan_check("scan_fwd", s));
    RST_REQUIRE(in && in->x && in->delta && in->A && in->B && in->C && y, "scan_fwd: null operand");
    Scan a{};
    scan_shape(&a, s, false);
    const size_t need = scan_carve(&a, nullptr, false);
    if (need && (workspace == nullptr || workspace_bytes < need))
        return fail(RST_ERR_WORKSPACE, "scan_fwd: workspace too small (%zu < %zu)", workspace_bytes, need);
    RST_REQUIRE(aligned16(workspace), "scan_fwd: workspace not aligned to 16 bytes");
    scan_carve(&a, static_cast<char*>(workspace), false);
    a.x = in->x; a.delta = in->delta; a.A = in->A; a.Bm = in->B; a.Cm = in->C; a.Dskip = in->D; a.z = in->z; a.dbias = in->delta_bias;
    a.h0 = state_in; a.y = y; a.last = state_out; a.ckpt = saved;
    const int W = scan_waves(a.N);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define FWD(T, W_) (a.z ? scan_fwd_t<T, W_, true>(a, st) : scan_fwd_t<T, W_, false>(a, st))
    return SCAN_TYPES(FWD);
#undef FWD
}

int rst_scan_bwd(const rst_scan_desc* s, const rst_scan_inputs* in, const float* saved, const void* dy, const float* dstate_out,
                 const rst_scan_grads* out, float* dstate_in, void* workspace, size_t workspace_bytes, void* stream) {
    RST_TRY(scan_check("scan_bwd", s));
    RST_REQUIRE(in && in->x && in->delta && in->A && in->B && in->C && saved && dy, "scan_bwd: null operand");
    RST_REQUIRE(out && out->x && out->delta && out->A && out->B && out->C && (!in->z || out->z), "scan_bwd: null gradient");
    Scan a{};
    scan_shape(&a, s, true);
    const size_t need = scan_carve(&a, nullptr, true);
    if (workspace == nullptr || workspace_bytes < need)
        return fail(RST_ERR_WORKSPACE, "scan_bwd: workspace too small (%zu < %zu)", workspace_bytes, need);
    RST_REQUIRE(aligned16(workspace), "scan_bwd: workspace not aligned to 16 bytes");
    scan_carve(&a, static_cast<char*>(workspace), true);
    a.x = in->x; a.delta = in->delta; a.A = in->A; a.Bm = in->B; a.Cm = in->C; a.Dskip = in->D; a.z = in->z; a.dbias = in->delta_bias;
    a.ckpt = const_cast<float*>(saved); a.dy = dy; a.dlast = dstate_out;
    a.dx = out->x; a.ddelta = out->delta; a.dB = out->B; a.dC = out->C; a.dz = out->z; a.dh0 = dstate_in;
    const int W = scan_waves(a.N);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define BWD(T, W_)                                                                                                      \
    (a.z ? scan_bwd_t<T, W_, true>(a, out->A, out->D, out->delta_bias, st) : scan_bwd_t<T, W_, false>(a, out->A, out->D, out->delta_bias, st))
    return SCAN_TYPES(BWD);
#undef BWD
}

int rst_scan_update(const rst_scan_desc* s, const rst_scan_inputs* in, const float* state_in, float* state_out, void* y, void* stream) {
    RST_TRY(scan_check("scan_update", s));
    RST_REQUIRE(s->L == 1, "scan_update: one token, not %lld", (long long)s->L);
    RST_REQUIRE(in && in->x && in->delta && in->A && in->B && in->C && y && state_in && state_out, "scan_update: null operand");
    const int W = scan_waves(s->N);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define UPD(T, NL) scan_update_t<T, NL>(s, in, state_in, state_out, static_cast<T*>(y), st)
    return SCAN_TYPES(UPD);
#undef UPD
}

}  // extern "C"
