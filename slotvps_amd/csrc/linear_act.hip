// Dense layer of 16-bit rows with bias, activation and residual in the product's epilogue, and its gradient:
//   y = act(x W^T + b) + r,   g = act'(x W^T + b)
//   dz = dy g,   dx = dz W,   dW = dz^T x,   db = column sums of dz   (the residual's gradient is dy itself)
//
// One product kernel serves all three: C[m, n] = sum_k X(m, k) W(n, k) with either operand stored k-contiguous ([m][k]) or k-major
// ([k][m]): forward (contiguous, contiguous), dx (contiguous, k-major), dW (k-major, k-major). Fragments of a k-contiguous tile are 16-byte
// LDS reads, of a k-major tile two hardware-transposed reads. Sums are fp32; bias, activation, slope and residual act on them before the
// one rounding of y. The slope g is stored instead of the pre-activation: held as int16 in units of 2^-14 it is off by 3e-5 (a 16-bit
// pre-activation in bf16: by up to 4e-3 times the curvature), and the backward pass needs no transcendental. That is absolute: a slope below
// 2^-7 is coarser than bf16's own rounding, below 2^-4 than fp16's, and GELU's below z = -4.7 is held as 0. dz is rounded to 16 bits once, as an
// operand of both products: with an activation dx and dW are 1.4 times as far off as their own rounding, without one dz is dy itself.
//
// Tile BM x BN x 64, WM x WN waves; operand tiles come by 16-byte LDS-DMA, the next ones while this one is multiplied. The W fragment is the
// MFMA's row operand: a lane owns one row m and four consecutive n per accumulator quad. Tiles behind each other in memory go to one XCD (its L2
// holds the shared operand rows). Few tiles: the k range is split over workgroups, fp32 partial sums are added in order (same epilogue).
//
// Operands whose rows do not start on 16 bytes or whose length is no multiple of 8 are first copied with zero-padded rows (linear_pack).
//
// Bound: matrix instructions, from about 1000 columns on; they run at the clock that the power allows (8192 cubed with operands of zeros:
// 600 us). Measured in bf16: 8192 cubed 786 us = 1399 TFLOP/s, dx 824 us, dW 861 us; 10240 x 6144 -> 1536 146 us = 1325 TFLOP/s. Narrower ones
// by their bytes and the epilogue: 32768 x 384 -> 1536 61 us, with GELU 80 us (13 vector and 2 transcendental instructions per value, which
// with one workgroup per CU nothing runs under). A few rows by the latency of one pass over the weights.
#include <type_traits>

#include "attention.h"
#include "../../include/slotvps_hip.h"

namespace svps {

enum { kActNone = 0, kActRelu = 1, kActGelu = 2 };

struct LinArgs {
    const void* x; const void* w;               // operands of the product
    long long ldx, ldw;                         // elements between rows of the STORED matrix
    int M, N, K, splits;
    const void* bias; int bias_f32;             // [N] or null
    const void* residual; void* y; void* gate;  // [M, N] contiguous; residual / gate may be null
    float* part; int ldp;                       // splits > 1: [splits][M][ldp]
    int act;
};

template <int BYTES> __device__ __forceinline__ int lin_swz(int row) {      // row of BYTES bytes
    if constexpr (BYTES >= 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return att_swz<BYTES / 2>(row);
}

// An operand's tile of one 64-deep step. KM = false: R rows (m or n side) x 64 k;  KM = true: 64 k rows x R columns.
// Every lane's offsets inside the tile are computed once; a step only moves the wave-uniform base. Rows (columns) behind the operand's
// end read its last ones again: they only reach accumulators that are not stored. What lies behind K must not count: the last step of a
// K that is no multiple of 64 takes zeros there.
template <int R, int NW, bool KM>
struct LinTile {
    static constexpr int LROWS = KM ? 64 : R, BYTES = KM ? R * 2 : 128, CH = BYTES / 16, RPP = 64 / CH, PIECES = LROWS / RPP, N = PIECES / NW;
    static_assert((CH & (CH - 1)) == 0 && CH <= 64, "the chunk swizzle permutes a power of two of chunks");
    static_assert(PIECES % NW == 0, "every wave stages the same number of pieces");
    const char* base;                           // of the tile at k = 0
    long long step;                             // bytes per step
    uint32_t off[N];
    __device__ __forceinline__ void init(const void* p, long long ld, int row0, int rows, int w, int lane) {
        base = (const char*)p + (KM ? (long long)row0 * 2 : (long long)row0 * ld * 2);
        step = KM ? 64 * ld * 2 : 128;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int lr = (i * NW + w) * RPP + lane / CH;
            const int chunk = (lane % CH) ^ lin_swz<BYTES>(lr);
            const int last = KM ? ((rows - 1 - row0) >> 3) : rows - 1 - row0;       // last chunk column / last row
            off[i] = KM ? (uint32_t)(lr * ld * 2) + (chunk < last ? chunk : last) * 16 : (uint32_t)((lr < last ? lr : last) * ld * 2) + chunk * 16;
        }
    }
    __device__ __forceinline__ void stage(int s, int K, char* lds, int w, int lane) const {
        const char* b = base + s * step;
        if ((s + 1) * 64 <= K) {
#pragma unroll
            for (int i = 0; i < N; ++i) dma_off(dma_base(b), off[i], lds + (i * NW + w) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int lr = (i * NW + w) * RPP + lane / CH;
                const int k = s * 64 + (KM ? lr : 8 * ((lane % CH) ^ lin_swz<BYTES>(lr)));
                dma_ptr(k < K ? b + off[i] : reinterpret_cast<const char*>(g_att_zero), lds + (i * NW + w) * 1024);
            }
        }
    }
};

template <typename T, int R, bool KM>
__device__ __forceinline__ typename AttVec<T>::v8 lin_frag(const char* lds, int row0, int ks, int lane) {
    typedef typename AttVec<T>::v8 v8;
    typedef typename AttVec<T>::v4 v4;
    if constexpr (!KM) {
        const int row = row0 + (lane & 31), h = lane >> 5;
        return *reinterpret_cast<const v8*>(lds + row * 128 + (((2 * ks + h) ^ lin_swz<128>(row)) << 4));
    } else {
        constexpr int BYTES = R * 2;
        const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
        const int ra = 16 * ks + 8 * (g >> 1) + q, rb = ra + 4;
        const int chunk = (row0 >> 3) + 2 * (g & 1) + (p >> 1);
        const char* pa = lds + ra * BYTES + ((chunk ^ lin_swz<BYTES>(ra)) << 4) + 8 * (p & 1);
        const char* pb = lds + rb * BYTES + ((chunk ^ lin_swz<BYTES>(rb)) << 4) + 8 * (p & 1);
        const v4 lo = ds_tr16((SVPS_LDS v4*)pa);
        const v4 hi = ds_tr16((SVPS_LDS v4*)pb);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// GELU through q = erfc(|z| / sqrt 2) / 2 in the form exp(-z^2 / 2) t P(t), t = 1 / (1 + p |z|) (the form of Abramowitz and Stegun 7.1.26),
// with the same exponential that the slope needs: one exponential and one reciprocal per value in place of erff's two branches
// (32768 x 384 -> 1536, when the whole took 96 us: 154 us with erff). P is of degree 5, a minimax fit over 0 <= |z| <= 15 whose error is bounded
// absolutely near 0 and relative to q behind: in fp32 arithmetic off by 2e-7 at most, and by 4.2e-5 of q at most down to |z| = 13 - far below
// zero q itself is the result, tiny but an ordinary number in bf16 (a fit of absolute error alone, one term shorter, is off by 1 % at z = -8).
template <int ACT>
__device__ __forceinline__ void lin_act(float z, float& y, float& g) {
    y = z;
    g = 1.f;
    if constexpr (ACT == kActRelu) {
        y = z > 0.f ? z : z != z ? z : 0.f;
        g = z > 0.f ? 1.f : z != z ? z : 0.f;
    } else if constexpr (ACT == kActGelu) {
        const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.295f, fabsf(z), 1.f));
        // z cdf(z) = max(z, 0) - |z| q
        const float q = e * t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.0836866647f, 0.25073567f), -0.053315904f), 0.15987511f), 0.108015954f), 0.118375756f);
        const float az = fminf(fabsf(z), 1e18f);                   // q and e are 0 long before: no infinity times zero
        y = fmaf(-az, q, fmaxf(z, 0.f));                           // (a NaN comes through q)
        g = z > 0.f ? 1.f - q : q;
        g = fmaf(copysignf(az, z) * 0.39894228040143268f, e, g);
    }
}

constexpr float kGateOne = 16384.f;               // slopes are held as int16 in units of 2^-14 (they lie in [-0.13, 1.13]): off by 3e-5 at most
constexpr short kGateNan = -32768;                // no slope: of a NaN
__device__ __forceinline__ short lin_gate(float g) { return g == g ? (short)(int)rintf(g * kGateOne) : kGateNan; }
__device__ __forceinline__ float lin_slope(short q) { return q == kGateNan ? NAN : (float)q * (1.f / kGateOne); }

template <typename T>
__device__ __forceinline__ float lin_bias(const LinArgs& a, int n) {
    return !a.bias ? 0.f : a.bias_f32 ? ((const float*)a.bias)[n] : (float)((const T*)a.bias)[n];
}
// of columns n, n + 1, ..: all on the way before the first is used. Columns behind the end take the last one's
template <typename T, int C>
__device__ __forceinline__ void lin_bias(const LinArgs& a, int n, float* b) {
#pragma unroll
    for (int j = 0; j < C; ++j) b[j] = 0.f;
    if (!a.bias) return;
    if (a.bias_f32) {
#pragma unroll
        for (int j = 0; j < C; ++j) b[j] = ((const float*)a.bias)[n + j < a.N ? n + j : a.N - 1];
    } else {
        T x[C];
#pragma unroll
        for (int j = 0; j < C; ++j) x[j] = ((const T*)a.bias)[n + j < a.N ? n + j : a.N - 1];
#pragma unroll
        for (int j = 0; j < C; ++j) b[j] = (float)x[j];
    }
}

// N8 consecutive columns n .. of row m (8: N % 8 == 0 and 16-byte aligned tensors; 1: any): their residual, asked for on its own so that a
// caller with several rows has all of them on the way before its first store (a load after a store waits for both; 40001 x 256 -> 333:
// 61 us row by row, 36 us so)
template <typename T, int N8> struct LinRow;
template <typename T> struct LinRow<T, 8> { typename AttVec<T>::v8 r; };
template <typename T> struct LinRow<T, 1> { T r[1]; };

template <typename T, int N8>
__device__ __forceinline__ LinRow<T, N8> lin_residual(const LinArgs& a, int m, int n) {
    return *reinterpret_cast<const LinRow<T, N8>*>((const T*)a.residual + (long long)m * a.N + n);
}

// and what becomes of their products z with the bias b
template <typename T, int N8, int ACT>
__device__ __forceinline__ void lin_epilogue(const LinArgs& a, int m, int n, const float* z, const float* b, const LinRow<T, N8>& res) {
    const long long o = (long long)m * a.N + n;
    float y[N8], g[N8];
#pragma unroll
    for (int j = 0; j < N8; ++j) {
        lin_act<ACT>(z[j] + b[j], y[j], g[j]);
        if (a.residual) y[j] += (float)res.r[j];
    }
    if constexpr (N8 == 8) {
        *reinterpret_cast<typename AttVec<T>::v8*>((T*)a.y + o) = att_pack<T>(y);
        if (a.gate) {
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            s16x8 q;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = lin_gate(g[j]);
            *reinterpret_cast<s16x8*>((short*)a.gate + o) = q;
        }
    } else {
        ((T*)a.y)[o] = (T)y[0];
        if (a.gate) ((short*)a.gate)[o] = lin_gate(g[0]);
    }
}

template <typename T, int N8>
__device__ __forceinline__ void lin_epilogue_any(const LinArgs& a, int m, int n, const float* z, const float* b) {
    LinRow<T, N8> res = {};
    if (a.residual) res = lin_residual<T, N8>(a, m, n);
    if (a.act == kActGelu) lin_epilogue<T, N8, kActGelu>(a, m, n, z, b, res);
    else if (a.act == kActRelu) lin_epilogue<T, N8, kActRelu>(a, m, n, z, b, res);
    else lin_epilogue<T, N8, kActNone>(a, m, n, z, b, res);
}

__device__ __forceinline__ bool lin_vec(const LinArgs& a) {
    return a.N % 8 == 0 && !(((uintptr_t)a.y | (uintptr_t)a.residual | (uintptr_t)a.gate) & 15);
}

template <typename T, int BM, int BN, int WM, int WN, bool XK, bool WK>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_kernel(LinArgs a) {
    typedef typename AttVec<T>::v8 v8;
    constexpr int NW = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32, XB = BM * 128, WB = BN * 128;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w / WN, wn = w - wm * WN;
    const int tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    // consecutive workgroups go round the 8 XCDs: XCD x takes the x-th eighth of the tile order, in which groups of 8 tile rows are walked
    // column by column - its resident tiles share few rows of either operand
    const int total = tm * tn;
    const int split = blockIdx.x / total;
    int id = blockIdx.x - split * total;
    {
        const int x = id & 7, q = id >> 3, per = total >> 3, rem = total & 7;
        id = x * per + (x < rem ? x : rem) + q;
    }
    const int per_group = 8 * tn, grp = id / per_group, in = id - grp * per_group;
    const int rows_in = tm - grp * 8 < 8 ? tm - grp * 8 : 8;
    const int m0 = (grp * 8 + in % rows_in) * BM, n0 = (in / rows_in) * BN;

    const int steps = (a.K + 63) / 64;
    int sb = 0, se = steps;
    if (a.splits > 1) {
        const int per = (steps + a.splits - 1) / a.splits;
        sb = split * per;
        se = sb + per < steps ? sb + per : steps;
    }
    LinTile<BM, NW, XK> tx;
    LinTile<BN, NW, WK> tw;
    tx.init(a.x, a.ldx, m0, a.M, w, lane);
    tw.init(a.w, a.ldw, n0, a.N, w, lane);
    f32x16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    v8 xf[2][MI], wf[2][NI];
    auto fetch = [&](const char* lx, const char* lw, int ks, int to) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NI; ++j) wf[to][j] = lin_frag<T, BN, WK>(lw, (wn * NI + j) * 32, ks, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i) xf[to][i] = lin_frag<T, BM, XK>(lx, (wm * MI + i) * 32, ks, lane);
    };
    auto multiply = [&](int from) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(wf[from][j], xf[from][i], acc[i][j]);
    };
    // (the scheduling fences keep reads, requests and products where they stand: left alone, the compiler sinks every read to just before
    // its use and waits for it there)
    auto fence = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
    if constexpr (NW == 8) {
        // One workgroup per CU, two waves per SIMD that take turns: while the first four multiply half a step (16 products, 512 cycles),
        // the others read their fragments of the next half and ask for operand tiles; then they change places, a barrier each time. A wave
        // held up by a request or a read never holds products up (8192 cubed: 810 us; both waves doing the same, the requests behind one
        // barrier per step, 935; the requests between a wave's own products 950).
        // LDS holds two tiles of w and three of x (160 KB). Phases: the first waves read tile s in 4 s and 4 s + 2, the second in 4 s + 1
        // and 4 s + 3, so its place is free from 4 s + 4 on. In step s the tiles w of s + 1 and x of s + 2 are asked for (phases 4 s, 4 s + 1
        // and 4 s + 2, 4 s + 3); before the barrier that ends 4 s + 3 every wave waits for its pieces of both tiles of s + 1, and only its
        // pieces of x of s + 2 stay in flight.
        const bool second = w >= 4;
        auto stage_x = [&](int s, int buf) __attribute__((always_inline)) { tx.stage(s, a.K, smem + buf * XB, w, lane); };
        auto stage_w = [&](int s) __attribute__((always_inline)) { tw.stage(s, a.K, smem + 3 * XB + ((s - sb) & 1) * WB, w, lane); };
        auto landed = [&](bool more) __attribute__((always_inline)) {
            if (more) wait_vm<decltype(tx)::N>();
            else wait_vm<0>();
        };
        if (sb < se) {
            stage_w(sb);
            stage_x(sb, 0);
            if (sb + 1 < se) stage_x(sb + 1, 1);
            landed(sb + 1 < se);
        }
        wg_barrier();
        if (second) wg_barrier();                                  // a phase behind
        int xb = 0;
        for (int s = sb; s < se; ++s) {
            const char* lx = smem + xb * XB;
            const char* lw = smem + 3 * XB + ((s - sb) & 1) * WB;
            auto half = [&](auto which) __attribute__((always_inline)) {
                constexpr int HALF = decltype(which)::value;
                auto ask = [&]() __attribute__((always_inline)) {
                    if (HALF == 0) {
                        if (s + 1 < se) stage_w(s + 1);
                    } else {
                        if (s + 2 < se) stage_x(s + 2, xb == 0 ? 2 : xb - 1);
                    }
                };
                // reads first; where both operands are read transposed (twice the reads) the requests (dW at 8192 cubed: 900 and 850 us;
                // the row-major product 810 and 825 us)
                if constexpr (XK && WK) {
                    ask();
                    fence();
                }
                fetch(lx, lw, 2 * HALF, 0);
                fetch(lx, lw, 2 * HALF + 1, 1);
                if constexpr (!(XK && WK)) ask();
                if (HALF == 1 && second) landed(s + 2 < se);
                fence();
                wg_barrier();
                fence();
                multiply(0);
                multiply(1);
                fence();
                if (HALF == 1 && !second) landed(s + 2 < se);
                wg_barrier();
                fence();
            };
            half(std::integral_constant<int, 0>{});
            half(std::integral_constant<int, 1>{});
            xb = xb == 2 ? 0 : xb + 1;
        }
        if (!second) wg_barrier();
    } else {
        // Several workgroups per CU overlap by themselves. Fragments are read one 16-deep slice ahead of the products. The barrier stands
        // BEFORE the last slice's products: by then the step's tile is in registers, so the tile after next may overwrite it, the next one
        // has had a step to arrive, and its first fragments are read under the last products.
        auto tile = [&](int s) __attribute__((always_inline)) { return smem + ((s - sb) & 1) * (XB + WB); };
        auto stage = [&](int s) __attribute__((always_inline)) {
            tx.stage(s, a.K, tile(s), w, lane);
            tw.stage(s, a.K, tile(s) + XB, w, lane);
        };
        auto read = [&](int s, int ks, int to) __attribute__((always_inline)) { fetch(tile(s), tile(s) + XB, ks, to); };
        auto products = [&](int from) __attribute__((always_inline)) {
            fence();
            multiply(from);
            fence();
        };
        if (sb < se) {
            stage(sb);
            wait_vm<0>();
            wg_barrier();
            if (sb + 1 < se) stage(sb + 1);
            read(sb, 0, 0);
        }
        for (int s = sb; s < se; ++s) {
            read(s, 1, 1);
            products(0);
            read(s, 2, 0);
            products(1);
            read(s, 3, 1);
            products(0);
            if (s + 1 < se) {
                wait_vm<0>();
                wg_barrier();
                if (s + 2 < se) stage(s + 2);
                read(s + 1, 0, 0);
            }
            products(1);
        }
    }
    // Epilogue: a wave turns its 32-row blocks around through its own piece of LDS, so that 8 lanes write 128 consecutive bytes of a row
    // (straight from the accumulators a lane would hold 4 columns of its own row: 32 rows per access, four times the cache-line visits).
    constexpr int COLS = NI * 32, LROW = COLS * 4 + 16;
    static_assert(NW * 32 * LROW <= 2 * (XB + WB), "the epilogue reuses the operand tiles");
    wg_barrier();                                                  // every wave has read its last operand tile
    char* my = smem + w * 32 * LROW;
    const bool vec = lin_vec(a);
    constexpr int LPR = COLS / 8, RPP = 64 / LPR;                  // lanes per row, rows per pass
    constexpr int RPL = 64 / COLS;                                 // rows per pass with a lane per column
    static_assert(COLS == 32 || COLS == 64, "a lane per column");
    float bias[8];                                                 // a lane's columns are the same in every pass
    if (a.splits == 1) lin_bias<T, 8>(a, n0 + wn * COLS + (vec ? (lane % LPR) * 8 : lane % COLS), bias);
    auto block = [&](auto which, auto act) __attribute__((always_inline)) {
        constexpr int i = decltype(which)::value, ACT = decltype(act)::value;
        const int mb = m0 + (wm * MI + i) * 32, nb = n0 + wn * COLS;
        if (mb >= a.M || nb >= a.N) return;
        auto turn = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
                    *reinterpret_cast<f32x4*>(my + r * LROW + (32 * j + 8 * g + 4 * h) * 4) = v;
                }
        };
        if (a.splits > 1 || vec) {
            const int c = (lane % LPR) * 8, n = nb + c;
            LinRow<T, 8> res[32 / RPP];
            if (a.residual && a.splits == 1 && n < a.N) {
#pragma unroll
                for (int q = 0; q < 32 / RPP; ++q) {
                    const int m = mb + q * RPP + lane / LPR;
                    res[q] = lin_residual<T, 8>(a, m < a.M ? m : a.M - 1, n);
                }
            }
            turn();
#pragma unroll
            for (int q = 0; q < 32 / RPP; ++q) {
                const int rr = q * RPP + lane / LPR, m = mb + rr;
                if (m < a.M && n < a.N) {
                    float z[8];
                    *reinterpret_cast<f32x4*>(z) = *reinterpret_cast<const f32x4*>(my + rr * LROW + c * 4);
                    *reinterpret_cast<f32x4*>(z + 4) = *reinterpret_cast<const f32x4*>(my + rr * LROW + c * 4 + 16);
                    if (a.splits > 1) {                            // ldp = N rounded up to 8
                        float* p = a.part + ((long long)split * a.M + m) * a.ldp + n;
                        *reinterpret_cast<f32x4*>(p) = f32x4{z[0], z[1], z[2], z[3]};
                        *reinterpret_cast<f32x4*>(p + 4) = f32x4{z[4], z[5], z[6], z[7]};
                    } else {
                        lin_epilogue<T, 8, ACT>(a, m, n, z, bias, res[q]);
                    }
                }
            }
        } else {                                                   // a lane per column
            const int cc = lane % COLS, n = nb + cc;
            turn();
            if (n >= a.N) return;
#pragma unroll 1
            for (int q0 = 0; q0 < 32 / RPL; q0 += 8) {             // written out eight rows at a time: all of them overrun the instruction cache
                LinRow<T, 1> res[8];
                if (a.residual) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int m = mb + (q0 + q) * RPL + lane / COLS;
                        res[q] = lin_residual<T, 1>(a, m < a.M ? m : a.M - 1, n);
                    }
                }
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const int rr = (q0 + q) * RPL + lane / COLS, m = mb + rr;
                    if (m < a.M) {
                        const float z = *reinterpret_cast<const float*>(my + rr * LROW + cc * 4);
                        lin_epilogue<T, 1, ACT>(a, m, n, &z, bias, res[q]);
                    }
                }
            }
        }
    };
    auto store = [&](auto act) __attribute__((always_inline)) {
        static_assert(MI == 1 || MI == 2 || MI == 4, "row blocks of a wave");
        block(std::integral_constant<int, 0>{}, act);
        if constexpr (MI > 1) block(std::integral_constant<int, 1>{}, act);
        if constexpr (MI > 2) {
            block(std::integral_constant<int, 2>{}, act);
            block(std::integral_constant<int, 3>{}, act);
        }
    };
    if (a.act == kActGelu) store(std::integral_constant<int, kActGelu>{});
    else if (a.act == kActRelu) store(std::integral_constant<int, kActRelu>{});
    else store(std::integral_constant<int, kActNone>{});
}

// the splits of a product added in order, then the same epilogue: 8 columns per thread
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(LinArgs a) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int cols = a.ldp >> 3;
    const long long m = id / cols;
    const int n = (int)(id - m * cols) * 8;
    if (m >= a.M) return;
    float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const f32x4* p = reinterpret_cast<const f32x4*>(a.part + ((long long)s * a.M + m) * a.ldp + n);
        const f32x4 u = p[0], v = p[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) { z[e] += u[e]; z[4 + e] += v[e]; }
    }
    float bias[8];
    lin_bias<T, 8>(a, n, bias);
    if (lin_vec(a)) {
        lin_epilogue_any<T, 8>(a, (int)m, n, z, bias);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < a.N) lin_epilogue_any<T, 1>(a, (int)m, n + j, z + j, bias + j);
    }
}

// Few rows (M <= 16 MT): a workgroup takes 16 columns, its 8 waves every eighth 32-deep slice of k; W goes from memory to the matrix operand
// without LDS (64 bytes of a row per lane group, each value once) with up to 4 slices of a wave in flight, the eight sums meet in LDS.
// Bound by the read of W; one launch, no partial sums in memory.
typedef float f32x4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4v mfma_16x16(bf16x8 a, bf16x8 b, f32x4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4v mfma_16x16(f16x8 a, f16x8 b, f32x4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <typename T, int MT>
__global__ __launch_bounds__(512) void linear_few_kernel(LinArgs a) {
    typedef typename AttVec<T>::v8 v8;
    __shared__ float red[8][MT][64][4];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16;
    const int nr = n0 + r < a.N ? n0 + r : a.N - 1;                // rows behind the end read the last one again: not stored
    const T* wp = (const T*)a.w + nr * a.ldw + 8 * q;
    const T* xp[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xp[t] = (const T*)a.x + (16 * t + r < a.M ? 16 * t + r : a.M - 1) * a.ldx + 8 * q;
    f32x4v acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4v{0.f, 0.f, 0.f, 0.f};
    const u32x4 zero = {0, 0, 0, 0};
    for (int k0 = 32 * w; k0 < a.K; k0 += 1024) {                  // K is a multiple of 8
        u32x4 wv[4], xv[4][MT];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = k0 + 256 * u;
            const bool in = k + 8 * q < a.K;
            wv[u] = zero;
            if (in) wv[u] = *reinterpret_cast<const u32x4*>(wp + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                xv[u][t] = zero;
                if (in) xv[u][t] = *reinterpret_cast<const u32x4*>(xp[t] + k);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = mfma_16x16(__builtin_bit_cast(v8, wv[u]), __builtin_bit_cast(v8, xv[u][t]), acc[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4v*>(red[w][t][lane]) = acc[t];
    __syncthreads();
    // lane (r, q) of a wave held row m = r and columns 4 q .. 4 q + 3 of its tile
    for (int o = threadIdx.x; o < 256 * MT; o += 512) {
        const int t = o >> 8, m = 16 * t + ((o >> 4) & 15), c = o & 15, n = n0 + c;
        if (m >= a.M || n >= a.N) continue;
        float z = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) z += red[k][t][(c >> 2) * 16 + ((o >> 4) & 15)][c & 3];
        const float b = lin_bias<T>(a, n);
        lin_epilogue_any<T, 1>(a, m, n, &z, &b);
    }
}

// [rows, cols] with row stride ld -> [rows, ldo], ldo = cols rounded up to 8, zeros behind cols; two matrices in one launch (the second may
// have no rows). 8 columns per thread.
struct LinPack { const uint16_t* src[2]; uint16_t* dst[2]; long long ld[2]; int rows[2], cols; unsigned first; };

__global__ __launch_bounds__(256) void linear_pack_kernel(LinPack a) {
    const int which = blockIdx.x >= a.first;
    const long long id = (long long)(blockIdx.x - (which ? a.first : 0)) * 256 + threadIdx.x;
    const int per = (a.cols + 7) >> 3;
    const long long row = id / per;
    if (row >= a.rows[which]) return;
    const int c0 = (int)(id - row * per) * 8;
    const uint16_t* src = a.src[which] + row * a.ld[which] + c0;
    union { uint16_t e[8]; u32x4 v; } o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.e[j] = c0 + j < a.cols ? src[j] : (uint16_t)0;
    *reinterpret_cast<u32x4*>(a.dst[which] + row * (per * 8) + c0) = o.v;
}

// dz = dy * gate (stored with row stride ldz, zero padded; skipped when dz is null) and the column sums of dz over a chunk of rows.
// Workgroup: CT threads x 8 columns of 256 / CT rows at a time, four rows per thread in flight. CT = 32 (512 bytes of a row) for many rows;
// CT = 4 for few, where 32-column workgroups are what fills the chip and the one chunk's sums are db (dz and sums of 500 x 2048: 7.5 us wide,
// 5.9 us narrow; of 10240 x 1536: 19 us wide, 78 us narrow).
template <typename T, int CT>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T* dy, long long ldy, const short* gate, T* dz, int ldz, float* sums, void* db, int db_f32,
                                                        int M, int N, int rows_per) {
    typedef typename AttVec<T>::v8 v8;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    constexpr int RT = 256 / CT, COLS = CT * 8;
    __shared__ float red[RT][COLS + 1];
    const int tx = threadIdx.x % CT, ty = threadIdx.x / CT;
    const int c0 = blockIdx.x * COLS + tx * 8;
    const int r1 = (int)min((long long)M, ((long long)blockIdx.y + 1) * rows_per);
    const bool vec = N % 8 == 0 && !(ldy & 7) && !(((uintptr_t)dy | (uintptr_t)gate) & 15);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c0 < N && vec) {
        for (int mb = blockIdx.y * rows_per + ty; mb < r1; mb += 4 * RT) {
            v8 d[4];
            s16x8 g[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const long long m = mb + RT * u < r1 ? mb + RT * u : mb;
                d[u] = *reinterpret_cast<const v8*>(dy + m * ldy + c0);
                if (gate) g[u] = *reinterpret_cast<const s16x8*>(gate + m * N + c0);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const long long m = mb + RT * u;
                if (m >= r1) break;
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = (float)d[u][j];
                    if (gate) v[j] *= lin_slope(g[u][j]);
                    s[j] += v[j];
                }
                if (dz) *reinterpret_cast<v8*>(dz + m * ldz + c0) = att_pack<T>(v);
            }
        }
    } else if (c0 < N) {
        for (int m = blockIdx.y * rows_per + ty; m < r1; m += RT) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = 0.f;
                if (c0 + j < N) {
                    v[j] = (float)dy[(long long)m * ldy + c0 + j];
                    if (gate) v[j] *= lin_slope(gate[(long long)m * N + c0 + j]);
                }
                s[j] += v[j];
            }
            if (dz) *reinterpret_cast<v8*>(dz + (long long)m * ldz + c0) = att_pack<T>(v);
        }
    }
    if (!sums && !db) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[ty][tx * 8 + j] = s[j];
    __syncthreads();
    const int c = blockIdx.x * COLS + threadIdx.x;
    if (threadIdx.x >= COLS || c >= N) return;
    float t = 0.f;
#pragma unroll 8
    for (int k = 0; k < RT; ++k) t += red[k][threadIdx.x];
    if (sums) sums[(long long)blockIdx.y * N + c] = t;
    else if (db_f32) ((float*)db)[c] = t;
    else ((T*)db)[c] = (T)t;
}

// db = the chunks' sums: a workgroup takes 32 columns, eight rows of threads add every eighth chunk, the eight sums meet in LDS
template <typename T>
__global__ __launch_bounds__(256) void linear_db_kernel(const float* sums, int chunks, int N, void* db, int db_f32) {
    __shared__ float red[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    float t = 0.f;
    if (c < N) {
#pragma unroll 8
        for (int k = ty; k < chunks; k += 8) t += sums[(long long)k * N + c];
    }
    red[ty][tx] = t;
    __syncthreads();
    if (ty || c >= N) return;
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][tx];
    if (db_f32) ((float*)db)[c] = t;
    else ((T*)db)[c] = (T)t;
}

static inline int round8(int x) { return (x + 7) & ~7; }
static inline bool lin_direct(const void* p, long long ld, int cols) { return !((uintptr_t)p & 15) && !(ld & 7) && !(cols & 7); }

struct LinPlan { int tile, splits; size_t part_bytes; };

// Tile (256, 128 or 64 square; one, two and four workgroups of them fit a CU) and split of the k range, by a model of the time in
// microseconds. Measured at k = 8192: a 64-deep step of a full CU takes 1.5, 0.68 and 0.36 per workgroup on it, of a workgroup alone on
// its CU 1.5, 0.9 and 0.6; start and epilogue 6, 4 and 3; a split's partial sums go to memory and back at 4 TB/s and cost a launch.
// (8192 cubed: 256 gives 778 us, 128 1045 us; 500 x 256 -> 2048 with GELU: 256 20 us, 128 8.8 us, 64 5.0 us; dW of 32768 rows, 384 -> 1536: 64
// without split 239 us, 128 with 14 parts 67.5 us, 256 with 21 parts, which it takes, 66 us; 32768 x 384 -> 1536 with GELU: 256, which it takes,
// 72 and 80 us on two cards, 128 72 and 76 us.)
static LinPlan linear_plan(int M, int N, int K) {
    static const int tile[3] = {256, 128, 64}, fit[3] = {1, 2, 4};
    static const double full[3] = {1.5, 0.68, 0.36}, alone[3] = {1.5, 0.9, 0.6}, fixed[3] = {6.0, 4.0, 3.0};
    const long long cus = svps_num_cus(), steps = (K + 63) / 64;
    LinPlan p = {64, 1, 0};
    double best = 0.0;
    for (int i = 0; i < 3; ++i) {
        const long long tiles = ((M + tile[i] - 1LL) / tile[i]) * ((N + tile[i] - 1LL) / tile[i]);
        for (int s = 1; s <= 32 && (s == 1 || steps / s >= 4); ++s) {
            const long long wgs = tiles * s, round = cus * fit[i], rest = wgs % round;
            const double depth = (double)((steps + s - 1) / s);
            auto one = [&](long long on) { const double t = on * full[i]; return depth * (t > alone[i] ? t : alone[i]) + fixed[i]; };
            const double t = (double)(wgs / round) * one(fit[i]) + (rest ? one((rest + cus - 1) / cus) : 0.0) +
                             (s > 1 ? 4.0 + (double)s * M * N * 8.0 / 4e6 : 0.0);
            if (best == 0.0 || t < best) { best = t; p.tile = tile[i]; p.splits = s; }
        }
    }
    p.part_bytes = p.splits > 1 ? (size_t)p.splits * M * round8(N) * sizeof(float) : 0;
    return p;
}

template <typename T, int BM, int BN, int WM, int WN, bool XK, bool WK>
static int linear_launch_tile(const LinArgs& a, hipStream_t stream) {
    constexpr int LDS = (2 * (BM + BN) + (WM * WN == 8 ? BM : 0)) * 128;
    static SvpsLdsAttr attr;
    const hipError_t e = attr.ensure((const void*)linear_kernel<T, BM, BN, WM, WN, XK, WK>, LDS);
    if (e != hipSuccess) return (int)e;
    const unsigned grid = (unsigned)(((a.M + BM - 1LL) / BM) * ((a.N + BN - 1LL) / BN) * a.splits);
    hipLaunchKernelGGL((linear_kernel<T, BM, BN, WM, WN, XK, WK>), dim3(grid), dim3(64 * WM * WN), LDS, stream, a);
    return (int)hipGetLastError();
}

template <typename T, bool XK, bool WK>
static int linear_launch(LinArgs a, const LinPlan& p, float* part, hipStream_t stream) {
    a.splits = p.splits;
    a.part = part;
    a.ldp = round8(a.N);
    const int rc = p.tile == 256 ? linear_launch_tile<T, 256, 256, 2, 4, XK, WK>(a, stream)
                 : p.tile == 128 ? linear_launch_tile<T, 128, 128, 2, 2, XK, WK>(a, stream) : linear_launch_tile<T, 64, 64, 2, 2, XK, WK>(a, stream);
    if (rc || p.splits == 1) return rc;
    const long long threads = (long long)a.M * (a.ldp >> 3);
    hipLaunchKernelGGL(linear_join_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

static int linear_pack(const void* src, long long ld, void* dst, int rows, const void* src2, long long ld2, void* dst2, int rows2, int cols, hipStream_t stream) {
    LinPack a = {{(const uint16_t*)src, (const uint16_t*)src2}, {(uint16_t*)dst, (uint16_t*)dst2}, {ld, ld2}, {rows, rows2}, cols, 0};
    const long long per = (cols + 7) >> 3, g0 = (rows * per + 255) / 256, g1 = (rows2 * per + 255) / 256;
    a.first = (unsigned)g0;
    hipLaunchKernelGGL(linear_pack_kernel, dim3((unsigned)(g0 + g1)), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

// Up to here one launch without a workspace (linear_few_kernel). Against tiles of 64, in us: 256 -> 2048: 17 rows 2.5 / 3.7, 64 rows 3.6 / 3.8;
// 1536 -> 1536: 32 rows 6.0 / 7.0, 64 rows 9.0 / 7.8; 6144 -> 1536: 17 rows 14.3 / 9.8, 64 rows 28.8 / 12.1. The bound looks at the rows alone
// and so is too high for sums of thousands.
constexpr int kFewRows = 64;

static bool linear_shape_ok(int M, int K, int N, long long ldx, long long ldw) {
    const long long big = 1LL << 30;
    // 256 rows of an operand stay inside 32-bit offsets
    if (M <= 0 || K <= 0 || N <= 0 || M > big || K >= 1 << 22 || N >= 1 << 22 || ldx < K || ldw < K || ldx >= 1 << 22 || ldw >= 1 << 22) return false;
    // workgroups, packed rows and 8-element groups of every launch fit 31 bits
    return ((M + 127LL) / 128) * ((N + 127LL) / 128) <= big / 64 && ((M + 127LL) / 128) * ((K + 127LL) / 128) <= big / 64 &&
           ((K + 127LL) / 128) * ((N + 127LL) / 128) <= big / 64;
}

// workspace of a pass: aligned sections in this order
static size_t sect(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// rows per chunk of the column sums: all of them where they are few, 64 otherwise (at most 32768 chunks)
static inline int dz_rows(int M) { return M <= 512 ? M : (M > 64 * 32768 ? (M + 32767) / 32768 : 64); }

}  // namespace svps

extern "C" size_t svps_linear_act_workspace_bytes(int M, int K, int N, long long ldx, long long ldw, int unaligned) {
    using namespace svps;
    if (!linear_shape_ok(M, K, N, ldx, ldw)) return 0;
    const bool px = unaligned || (ldx & 7) || (K & 7), pw = unaligned || (ldw & 7) || (K & 7);
    return (px ? sect((size_t)M * round8(K) * 2) : 0) + (pw ? sect((size_t)N * round8(K) * 2) : 0) + (M <= kFewRows ? 0 : sect(linear_plan(M, N, K).part_bytes));
}

template <typename T>
static int linear_fwd_t(svps::LinArgs a, char* ws, hipStream_t s) {
    using namespace svps;
    const bool px = !lin_direct(a.x, a.ldx, a.K), pw = !lin_direct(a.w, a.ldw, a.K);
    const int k8 = round8(a.K);
    if (px || pw) {
        char* xs = ws;
        char* wsp = ws + (px ? sect((size_t)a.M * k8 * 2) : 0);
        const int rc = linear_pack(a.x, a.ldx, xs, px ? a.M : 0, a.w, a.ldw, wsp, pw ? a.N : 0, a.K, s);
        if (rc) return rc;
        if (px) { a.x = xs; a.ldx = k8; }
        if (pw) { a.w = wsp; a.ldw = k8; }
        ws = wsp + (pw ? sect((size_t)a.N * k8 * 2) : 0);
    }
    const int M = a.M, K = a.K;
    a.K = k8;
    if (M <= kFewRows) {
        const dim3 grid((a.N + 15) / 16), block(512);
        if (M <= 16) hipLaunchKernelGGL((linear_few_kernel<T, 1>), grid, block, 0, s, a);
        else if (M <= 32) hipLaunchKernelGGL((linear_few_kernel<T, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((linear_few_kernel<T, 4>), grid, block, 0, s, a);
        return (int)hipGetLastError();
    }
    return linear_launch<T, false, false>(a, linear_plan(M, a.N, K), (float*)ws, s);
}

extern "C" int svps_linear_act_fwd(const void* x, long long ldx, const void* w, long long ldw, const void* bias, int bias_f32, const void* residual,
                                   int act, void* y, void* gate, void* workspace, size_t workspace_bytes, int M, int K, int N, int dtype, void* stream) {
    using namespace svps;
    if (!x || !w || !y) return SVPS_ERR_BAD_ARG;
    if (act < kActNone || act > kActGelu || (dtype != SVPS_DTYPE_BF16 && dtype != SVPS_DTYPE_F16)) return SVPS_ERR_BAD_ARG;
    if (!linear_shape_ok(M, K, N, ldx, ldw)) return SVPS_ERR_BAD_SHAPE;
    const size_t need = (lin_direct(x, ldx, K) ? 0 : sect((size_t)M * round8(K) * 2)) + (lin_direct(w, ldw, K) ? 0 : sect((size_t)N * round8(K) * 2)) +
                        (M <= kFewRows ? 0 : sect(linear_plan(M, N, K).part_bytes));
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return SVPS_ERR_WORKSPACE;
    LinArgs a = {};
    a.x = x; a.w = w; a.ldx = ldx; a.ldw = ldw; a.M = M; a.N = N; a.K = K;
    a.bias = bias; a.bias_f32 = bias_f32; a.residual = residual; a.y = y; a.gate = gate; a.act = act;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SVPS_DTYPE_BF16 ? linear_fwd_t<__bf16>(a, (char*)workspace, s) : linear_fwd_t<_Float16>(a, (char*)workspace, s);
}

namespace svps {
struct LinBwdPlan { size_t dz, x, w, sums, part; int chunks; };
static LinBwdPlan linear_bwd_plan(int M, int K, int N, bool own_dz, bool pack_x, bool pack_w, bool dx, bool dw, bool db) {
    LinBwdPlan p;
    p.chunks = (M + dz_rows(M) - 1) / dz_rows(M);
    p.dz = own_dz ? sect((size_t)M * round8(N) * 2) : 0;
    p.x = dw && pack_x ? sect((size_t)M * round8(K) * 2) : 0;
    p.w = dx && pack_w ? sect((size_t)N * round8(K) * 2) : 0;
    p.sums = db && p.chunks > 1 ? sect((size_t)p.chunks * N * sizeof(float)) : 0;
    const size_t a = dx ? linear_plan(M, K, N).part_bytes : 0, b = dw ? linear_plan(N, K, M).part_bytes : 0;
    p.part = sect(a > b ? a : b);                                  // one after the other on one stream: shared
    return p;
}

template <typename T>
static int linear_bwd_t(const T* dy, long long ldy, const T* x, long long ldx, const T* w, long long ldw, const short* gate, T* dx, T* dw, void* db,
                        int db_f32, char* ws, const LinBwdPlan& p, int M, int K, int N, hipStream_t s) {
    int rc;
    const T* dz = dy;
    long long ldz = ldy;
    T* own = nullptr;
    if (p.dz) {
        own = (T*)ws;
        dz = own;
        ldz = round8(N);
        ws += p.dz;
    }
    char* xs = ws; ws += p.x;
    char* wsp = ws; ws += p.w;
    float* sums = p.sums ? (float*)ws : nullptr; ws += p.sums;
    float* part = (float*)ws;
    if (own || db) {
        if (p.chunks == 1)
            hipLaunchKernelGGL((linear_dz_kernel<T, 4>), dim3((N + 31) / 32, 1), dim3(256), 0, s, dy, ldy, gate, own, (int)ldz, sums, db, db_f32, M, N, M);
        else
            hipLaunchKernelGGL((linear_dz_kernel<T, 32>), dim3((N + 255) / 256, p.chunks), dim3(256), 0, s, dy, ldy, gate, own, (int)ldz, sums, db, db_f32, M, N, dz_rows(M));
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
        if (sums) {
            hipLaunchKernelGGL(linear_db_kernel<T>, dim3((N + 31) / 32), dim3(256), 0, s, sums, p.chunks, N, db, db_f32);
            e = hipGetLastError();
            if (e != hipSuccess) return (int)e;
        }
    }
    if (p.w || p.x) {
        if ((rc = linear_pack(x, ldx, xs, p.x ? M : 0, w, ldw, wsp, p.w ? N : 0, K, s))) return rc;
    }
    if (dx) {                                                      // dx[m, k] = sum_n dz[m, n] W[n, k]
        LinArgs a = {};
        a.x = dz; a.ldx = ldz; a.w = w; a.ldw = ldw; a.M = M; a.N = K; a.K = N; a.y = dx;
        if (p.w) {
            a.w = wsp;
            a.ldw = round8(K);
        }
        if ((rc = linear_launch<T, false, true>(a, linear_plan(M, K, N), part, s))) return rc;
    }
    if (dw) {                                                      // dW[n, k] = sum_m dz[m, n] x[m, k]
        LinArgs a = {};
        a.x = dz; a.ldx = ldz; a.w = x; a.ldw = ldx; a.M = N; a.N = K; a.K = M; a.y = dw;
        if (p.x) {
            a.w = xs;
            a.ldw = round8(K);
        }
        if ((rc = linear_launch<T, true, true>(a, linear_plan(N, K, M), part, s))) return rc;
    }
    return 0;
}
}  // namespace svps

extern "C" size_t svps_linear_act_bwd_workspace_bytes(int M, int K, int N, long long ldy, long long ldx, long long ldw, int unaligned, int has_gate,
                                                      int want_dx, int want_dw, int want_db) {
    using namespace svps;
    if (!linear_shape_ok(M, K, N, ldx, ldw) || ldy < N || ldy >= 1 << 22) return 0;
    const LinBwdPlan p = linear_bwd_plan(M, K, N, has_gate || unaligned || (ldy & 7) || (N & 7), unaligned || (ldx & 7) || (K & 7),
                                         unaligned || (ldw & 7) || (K & 7), want_dx, want_dw, want_db);
    return p.dz + p.x + p.w + p.sums + p.part;
}

extern "C" int svps_linear_act_bwd(const void* dy, long long ldy, const void* x, long long ldx, const void* w, long long ldw, const void* gate,
                                   void* dx, void* dw, void* db, int db_f32, void* workspace, size_t workspace_bytes, int M, int K, int N, int dtype,
                                   void* stream) {
    using namespace svps;
    if (!dy || (!dx && !dw && !db) || (dx && !w) || (dw && !x)) return SVPS_ERR_BAD_ARG;
    if (dtype != SVPS_DTYPE_BF16 && dtype != SVPS_DTYPE_F16) return SVPS_ERR_BAD_ARG;
    if (!linear_shape_ok(M, K, N, x ? ldx : K, w ? ldw : K) || ldy < N || ldy >= 1 << 22) return SVPS_ERR_BAD_SHAPE;
    const LinBwdPlan p = linear_bwd_plan(M, K, N, (dx || dw) && (gate || !lin_direct(dy, ldy, N)), !lin_direct(x, ldx, K), !lin_direct(w, ldw, K),
                                         dx != nullptr, dw != nullptr, db != nullptr);
    const size_t need = p.dz + p.x + p.w + p.sums + p.part;
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return SVPS_ERR_WORKSPACE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == SVPS_DTYPE_BF16)
        return linear_bwd_t<__bf16>((const __bf16*)dy, ldy, (const __bf16*)x, ldx, (const __bf16*)w, ldw, (const short*)gate, (__bf16*)dx, (__bf16*)dw,
                                    db, db_f32, (char*)workspace, p, M, K, N, s);
    return linear_bwd_t<_Float16>((const _Float16*)dy, ldy, (const _Float16*)x, ldx, (const _Float16*)w, ldw, (const short*)gate, (_Float16*)dx,
                                  (_Float16*)dw, db, db_f32, (char*)workspace, p, M, K, N, s);
}
