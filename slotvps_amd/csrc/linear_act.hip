// Dense layer of 16-bit rows with bias, activation and residual in the product's epilogue, and its gradient:
//   y = act(x W^T + b) + r,   g = act'(x W^T + b)
//   dz = dy g,   dx = dz W,   dW = dz^T x,   db = column sums of dz   (the residual's gradient is dy itself)
//
// One product kernel serves all three: C[m, n] = sum_k X(m, k) W(n, k) with either operand stored k-contiguous ([m][k]) or k-major
// ([k][m]): forward (contiguous, contiguous), dx (contiguous, k-major), dW (k-major, k-major). Fragments of a k-contiguous tile are 16-byte
// LDS reads, of a k-major tile two hardware-transposed reads. Sums are fp32; bias, activation, slope and residual act on them before the
// one rounding of y. The slope g is stored instead of the pre-activation: rounded once it is off by half a step, where the slope of a
// rounded pre-activation would be off by the rounding times the curvature, and the backward pass needs no transcendental.
//
// Tile BM x BN x 64, WM x WN waves; LDS double-buffered by 16-byte LDS-DMA, one barrier per 64-deep step. The W fragment is the MFMA's row
// operand: a lane owns one row m and four consecutive n per accumulator quad. Tiles behind each other in memory go to one XCD (its L2
// holds the shared operand rows). Few tiles: the k range is split over workgroups, fp32 partial sums are added in order (same epilogue).
//
// Operands whose rows do not start on 16 bytes or whose length is no multiple of 8 are first copied with zero-padded rows (linear_pack).
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

// KM = false: tile of `R` rows x 64 k (row0 .. on the m / n side);  KM = true: tile of 64 k rows x R columns
template <int R, int NW, bool KM>
__device__ __forceinline__ void lin_stage(const char* base, long long ld, int row0, int rows, int k0, int K, char* lds, int w, int lane) {
    constexpr int LROWS = KM ? 64 : R, BYTES = KM ? R * 2 : 128, CH = BYTES / 16, RPP = 64 / CH, PIECES = LROWS / RPP;
#pragma unroll
    for (int i = 0; i < (PIECES + NW - 1) / NW; ++i) {
        const int j = i * NW + w;
        if (PIECES % NW == 0 || j < PIECES) {
            const int lr = j * RPP + lane / CH;
            const int chunk = (lane % CH) ^ lin_swz<BYTES>(lr);
            const int sr = (KM ? k0 : row0) + lr, sc = (KM ? row0 : k0) + chunk * 8;     // stored row, column
            const bool ok = KM ? (sr < K && sc < rows) : (sr < rows && sc < K);
            dma16(ok ? base + ((long long)sr * ld + sc) * 2 : reinterpret_cast<const char*>(g_att_zero), lds + j * 1024);
        }
    }
}

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

__device__ __forceinline__ void lin_act(int act, float z, float& y, float& g) {
    y = z;
    g = 1.f;
    if (act == kActRelu) {
        y = fmaxf(z, 0.f);
        g = z > 0.f ? 1.f : 0.f;
        if (z != z) { y = z; g = z; }
    } else if (act == kActGelu) {
        const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
        y = z * cdf;
        g = cdf + z * 0.39894228040143268f * __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
    }
}

// four consecutive columns n .. n + 3 of row m
template <typename T>
__device__ __forceinline__ void lin_epilogue(const LinArgs& a, int m, int n, const float* z, bool vec) {
    typedef typename AttVec<T>::v4 v4;
    const long long o = (long long)m * a.N + n;
    float y[4], g[4];
    if (vec) {                                                   // N % 4 == 0, 8-byte aligned tensors
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.bias) {
            if (a.bias_f32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = ((const float*)a.bias)[n + j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = (float)((const T*)a.bias)[n + j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) lin_act(a.act, z[j] + b[j], y[j], g[j]);
        if (a.residual) {
            const v4 r = *reinterpret_cast<const v4*>((const T*)a.residual + o);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] += (float)r[j];
        }
        v4 yo, go;
#pragma unroll
        for (int j = 0; j < 4; ++j) { yo[j] = (T)y[j]; go[j] = (T)g[j]; }
        *reinterpret_cast<v4*>((T*)a.y + o) = yo;
        if (a.gate) *reinterpret_cast<v4*>((T*)a.gate + o) = go;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n + j >= a.N) break;
        const float b = !a.bias ? 0.f : a.bias_f32 ? ((const float*)a.bias)[n + j] : (float)((const T*)a.bias)[n + j];
        lin_act(a.act, z[j] + b, y[j], g[j]);
        if (a.residual) y[j] += (float)((const T*)a.residual)[o + j];
        ((T*)a.y)[o + j] = (T)y[j];
        if (a.gate) ((T*)a.gate)[o + j] = (T)g[j];
    }
}

__device__ __forceinline__ bool lin_vec(const LinArgs& a) {
    return a.N % 4 == 0 && !(((uintptr_t)a.y | (uintptr_t)a.residual | (uintptr_t)a.gate) & 7);
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
    const char* xb = (const char*)a.x;
    const char* wb = (const char*)a.w;
    auto stage = [&](int s, int buf) {
        char* l = smem + buf * (XB + WB);
        lin_stage<BM, NW, XK>(xb, a.ldx, m0, a.M, s * 64, a.K, l, w, lane);
        lin_stage<BN, NW, WK>(wb, a.ldw, n0, a.N, s * 64, a.K, l + XB, w, lane);
    };
    f32x16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    if (sb < se) stage(sb, 0);
    for (int s = sb; s < se; ++s) {
        const int buf = (s - sb) & 1;
        wait_vm<0>();
        wg_barrier();
        if (s + 1 < se) stage(s + 1, buf ^ 1);
        const char* lx = smem + buf * (XB + WB);
        const char* lw = lx + XB;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            v8 xf[MI], wf[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) xf[i] = lin_frag<T, BM, XK>(lx, (wm * MI + i) * 32, ks, lane);
#pragma unroll
            for (int j = 0; j < NI; ++j) wf[j] = lin_frag<T, BN, WK>(lw, (wn * NI + j) * 32, ks, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(wf[j], xf[i], acc[i][j]);
        }
    }
    const bool vec = lin_vec(a);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int m = m0 + (wm * MI + i) * 32 + r;
        if (m >= a.M) continue;
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = n0 + (wn * NI + j) * 32 + 8 * g + 4 * h;
                if (n >= a.N) continue;
                float z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = acc[i][j][4 * g + e];
                if (a.splits > 1) *reinterpret_cast<f32x4*>(a.part + ((long long)split * a.M + m) * a.ldp + n) = f32x4{z[0], z[1], z[2], z[3]};
                else lin_epilogue<T>(a, m, n, z, vec);
            }
    }
}

// the splits of a product added in order, then the same epilogue
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(LinArgs a) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int cols = a.ldp >> 2;
    const long long m = id / cols;
    const int n = (int)(id - m * cols) * 4;
    if (m >= a.M || n >= a.N) return;
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + ((long long)s * a.M + m) * a.ldp + n);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] += v[e];
    }
    lin_epilogue<T>(a, (int)m, n, z, lin_vec(a));
}

// [rows, cols] with row stride ld -> [rows, ldo], ldo = cols rounded up to 8, zeros behind cols. 8 columns per thread.
__global__ __launch_bounds__(256) void linear_pack_kernel(const uint16_t* src, long long ld, uint16_t* dst, int rows, int cols, int ldo) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int per = ldo >> 3;
    const long long row = id / per;
    if (row >= rows) return;
    const int c0 = (int)(id - row * per) * 8;
    union { uint16_t e[8]; u32x4 v; } o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.e[j] = c0 + j < cols ? src[row * ld + c0 + j] : (uint16_t)0;
    *reinterpret_cast<u32x4*>(dst + row * ldo + c0) = o.v;
}

// dz = dy * gate (stored with row stride ldz, zero padded; skipped when dz is null) and the column sums of dz over a chunk of rows.
// Workgroup: 256 columns (32 threads x 8) x 8 rows at a time over `rows_per` rows.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T* dy, long long ldy, const T* gate, T* dz, int ldz, float* sums, int M, int N, int rows_per) {
    typedef typename AttVec<T>::v8 v8;
    __shared__ float red[8][256];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c0 = blockIdx.x * 256 + tx * 8;
    const int r1 = (int)min((long long)M, ((long long)blockIdx.y + 1) * rows_per);
    const bool vec = N % 8 == 0 && !(ldy & 7) && !(((uintptr_t)dy | (uintptr_t)gate) & 15);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int m = blockIdx.y * rows_per + ty; m < r1; m += 8) {
        if (c0 >= N) break;
        float v[8];
        if (vec) {
            const v8 d = *reinterpret_cast<const v8*>(dy + (long long)m * ldy + c0);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)d[j];
            if (gate) {
                const v8 g = *reinterpret_cast<const v8*>(gate + (long long)m * N + c0);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= (float)g[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = 0.f;
                if (c0 + j < N) {
                    v[j] = (float)dy[(long long)m * ldy + c0 + j];
                    if (gate) v[j] *= (float)gate[(long long)m * N + c0 + j];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += v[j];
        if (dz) *reinterpret_cast<v8*>(dz + (long long)m * ldz + c0) = att_pack<T>(v);
    }
    if (!sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[ty][tx * 8 + j] = s[j];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][threadIdx.x];
    if (c < N) sums[(long long)blockIdx.y * N + c] = t;
}

template <typename T>
__global__ __launch_bounds__(256) void linear_db_kernel(const float* sums, int chunks, int N, void* db, int db_f32) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float t = 0.f;
    for (int k = 0; k < chunks; ++k) t += sums[(long long)k * N + c];
    if (db_f32) ((float*)db)[c] = t;
    else ((T*)db)[c] = (T)t;
}

static inline int round8(int x) { return (x + 7) & ~7; }
static inline bool lin_direct(const void* p, long long ld, int cols) { return !((uintptr_t)p & 15) && !(ld & 7) && !(cols & 7); }

struct LinPlan { int splits; size_t part_bytes; };

static LinPlan linear_plan(int M, int N, int K) {
    LinPlan p;
    const long long tiles = ((M + 127LL) / 128) * ((N + 127LL) / 128), want = 2LL * svps_num_cus();
    long long s = tiles * 2 > want ? 1 : want / tiles;
    const long long steps = (K + 63) / 64;
    if (s > steps / 2) s = steps / 2;
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    p.part_bytes = p.splits > 1 ? (size_t)p.splits * M * round8(N) * sizeof(float) : 0;
    return p;
}

template <typename T, bool XK, bool WK>
static int linear_launch(LinArgs a, const LinPlan& p, float* part, hipStream_t stream) {
    constexpr int BM = 128, BN = 128, WM = 2, WN = 2, LDS = 2 * (BM + BN) * 128;
    static SvpsLdsAttr attr;
    hipError_t e = attr.ensure((const void*)linear_kernel<T, BM, BN, WM, WN, XK, WK>, LDS);
    if (e != hipSuccess) return (int)e;
    a.splits = p.splits;
    a.part = part;
    a.ldp = round8(a.N);
    const unsigned grid = (unsigned)(((a.M + BM - 1LL) / BM) * ((a.N + BN - 1LL) / BN) * p.splits);
    hipLaunchKernelGGL((linear_kernel<T, BM, BN, WM, WN, XK, WK>), dim3(grid), dim3(64 * WM * WN), LDS, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return (int)e;
    const long long threads = (long long)a.M * (a.ldp >> 2);
    hipLaunchKernelGGL(linear_join_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

static int linear_pack(const void* src, long long ld, void* dst, int rows, int cols, hipStream_t stream) {
    const long long threads = (long long)rows * (round8(cols) >> 3);
    hipLaunchKernelGGL(linear_pack_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, (const uint16_t*)src, ld, (uint16_t*)dst, rows, cols, round8(cols));
    return (int)hipGetLastError();
}

static bool linear_shape_ok(int M, int K, int N, long long ldx, long long ldw) {
    const long long big = 1LL << 30;
    if (M <= 0 || K <= 0 || N <= 0 || M > big || K > big || N > big || ldx < K || ldw < K) return false;
    // workgroups, packed rows and 8-element groups of every launch fit 31 bits
    return ((M + 127LL) / 128) * ((N + 127LL) / 128) <= big / 64 && ((M + 127LL) / 128) * ((K + 127LL) / 128) <= big / 64 &&
           ((K + 127LL) / 128) * ((N + 127LL) / 128) <= big / 64;
}

// workspace of a pass: aligned sections in this order
static size_t sect(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

constexpr int kDzRows = 64;

}  // namespace svps

extern "C" size_t svps_linear_act_workspace_bytes(int M, int K, int N, long long ldx, long long ldw, int unaligned) {
    using namespace svps;
    if (!linear_shape_ok(M, K, N, ldx, ldw)) return 0;
    const bool px = unaligned || (ldx & 7) || (K & 7), pw = unaligned || (ldw & 7) || (K & 7);
    return (px ? sect((size_t)M * round8(K) * 2) : 0) + (pw ? sect((size_t)N * round8(K) * 2) : 0) + sect(linear_plan(M, N, K).part_bytes);
}

template <typename T>
static int linear_fwd_t(svps::LinArgs a, char* ws, hipStream_t s) {
    using namespace svps;
    const LinPlan p = linear_plan(a.M, a.N, a.K);
    int rc;
    if (!lin_direct(a.x, a.ldx, a.K)) {
        if ((rc = linear_pack(a.x, a.ldx, ws, a.M, a.K, s))) return rc;
        a.x = ws;
        a.ldx = round8(a.K);
        ws += sect((size_t)a.M * a.ldx * 2);
    }
    if (!lin_direct(a.w, a.ldw, a.K)) {
        if ((rc = linear_pack(a.w, a.ldw, ws, a.N, a.K, s))) return rc;
        a.w = ws;
        a.ldw = round8(a.K);
        ws += sect((size_t)a.N * a.ldw * 2);
    }
    a.K = round8(a.K);
    return linear_launch<T, false, false>(a, p, (float*)ws, s);
}

extern "C" int svps_linear_act_fwd(const void* x, long long ldx, const void* w, long long ldw, const void* bias, int bias_f32, const void* residual,
                                   int act, void* y, void* gate, void* workspace, size_t workspace_bytes, int M, int K, int N, int dtype, void* stream) {
    using namespace svps;
    if (!x || !w || !y) return SVPS_ERR_BAD_ARG;
    if (act < kActNone || act > kActGelu || (dtype != SVPS_DTYPE_BF16 && dtype != SVPS_DTYPE_F16)) return SVPS_ERR_BAD_ARG;
    if (!linear_shape_ok(M, K, N, ldx, ldw)) return SVPS_ERR_BAD_SHAPE;
    const size_t need = (lin_direct(x, ldx, K) ? 0 : sect((size_t)M * round8(K) * 2)) + (lin_direct(w, ldw, K) ? 0 : sect((size_t)N * round8(K) * 2)) +
                        sect(linear_plan(M, N, K).part_bytes);
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
    p.chunks = (M + kDzRows - 1) / kDzRows;
    p.dz = own_dz ? sect((size_t)M * round8(N) * 2) : 0;
    p.x = dw && pack_x ? sect((size_t)M * round8(K) * 2) : 0;
    p.w = dx && pack_w ? sect((size_t)N * round8(K) * 2) : 0;
    p.sums = db ? sect((size_t)p.chunks * N * sizeof(float)) : 0;
    const size_t a = dx ? linear_plan(M, K, N).part_bytes : 0, b = dw ? linear_plan(N, K, M).part_bytes : 0;
    p.part = sect(a > b ? a : b);                                  // one after the other on one stream: shared
    return p;
}

template <typename T>
static int linear_bwd_t(const T* dy, long long ldy, const T* x, long long ldx, const T* w, long long ldw, const T* gate, T* dx, T* dw, void* db,
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
    if (own || sums) {
        // rows in chunks of kDzRows: few enough rows per workgroup to fill the chip, and the sums of a chunk are one fp32 row
        hipLaunchKernelGGL(linear_dz_kernel<T>, dim3((N + 255) / 256, p.chunks), dim3(256), 0, s, dy, ldy, gate, own, (int)ldz, sums, M, N, kDzRows);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
        if (sums) {
            hipLaunchKernelGGL(linear_db_kernel<T>, dim3((N + 255) / 256), dim3(256), 0, s, sums, p.chunks, N, db, db_f32);
            e = hipGetLastError();
            if (e != hipSuccess) return (int)e;
        }
    }
    if (dx) {                                                      // dx[m, k] = sum_n dz[m, n] W[n, k]
        LinArgs a = {};
        a.x = dz; a.ldx = ldz; a.w = w; a.ldw = ldw; a.M = M; a.N = K; a.K = N; a.y = dx;
        if (p.w) {
            if ((rc = linear_pack(w, ldw, wsp, N, K, s))) return rc;
            a.w = wsp;
            a.ldw = round8(K);
        }
        if ((rc = linear_launch<T, false, true>(a, linear_plan(M, K, N), part, s))) return rc;
    }
    if (dw) {                                                      // dW[n, k] = sum_m dz[m, n] x[m, k]
        LinArgs a = {};
        a.x = dz; a.ldx = ldz; a.w = x; a.ldw = ldx; a.M = N; a.N = K; a.K = M; a.y = dw;
        if (p.x) {
            if ((rc = linear_pack(x, ldx, xs, M, K, s))) return rc;
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
    if (!linear_shape_ok(M, K, N, ldx, ldw) || ldy < N) return 0;
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
    if (!linear_shape_ok(M, K, N, x ? ldx : K, w ? ldw : K) || ldy < N) return SVPS_ERR_BAD_SHAPE;
    if ((M + kDzRows - 1) / kDzRows > 65535) return SVPS_ERR_BAD_SHAPE;
    const LinBwdPlan p = linear_bwd_plan(M, K, N, (dx || dw) && (gate || !lin_direct(dy, ldy, N)), !lin_direct(x, ldx, K), !lin_direct(w, ldw, K),
                                         dx != nullptr, dw != nullptr, db != nullptr);
    const size_t need = p.dz + p.x + p.w + p.sums + p.part;
    if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return SVPS_ERR_WORKSPACE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == SVPS_DTYPE_BF16)
        return linear_bwd_t<__bf16>((const __bf16*)dy, ldy, (const __bf16*)x, ldx, (const __bf16*)w, ldw, (const __bf16*)gate, (__bf16*)dx, (__bf16*)dw,
                                    db, db_f32, (char*)workspace, p, M, K, N, s);
    return linear_bwd_t<_Float16>((const _Float16*)dy, ldy, (const _Float16*)x, ldx, (const _Float16*)w, ldw, (const _Float16*)gate, (_Float16*)dx,
                                  (_Float16*)dw, db, db_f32, (char*)workspace, p, M, K, N, s);
}
