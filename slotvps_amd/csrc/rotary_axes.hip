// Rotary positions with several axes (frame, row, column, ...) for queries and keys of clip tokens.
//
// Mathematics: the first R channels of a head are R / 2 pairs; pair j belongs to one axis a(j) and turns by
//     angle = p[n, a(j)] * f_j,   y1 = x1 cos - x2 sin,   y2 = x2 cos + x1 sin
// the other D - R channels pass. The gradient of a rotation is the rotation by the negative angle: the same kernel with `sign` = -1.
//
// Angles: p * f_j in float64 TURNS (f_j is handed over divided by 2 pi, in float64), reduced to a quarter turn there, and only the
// remainder - at most an eighth of a turn either way, exact to 2^-27 turns - goes to fp32 sine and cosine. In fp32 the product itself
// would be off by 6e-3 radians at position 1e5.
//
// Bound: bandwidth (each value read once, written once; 6 operations per pair). A work item is (token, 16 bytes of a head): it computes
// the cosines and sines of its pairs ONCE and walks over the heads of both tensors with them in registers, so the transcendental work is
// divided by the number of heads. Few tokens: the heads are dealt over grid.y instead, one launch either way.
#include "common.h"
#include "../../include/slotvps_hip.h"

namespace svps {

constexpr int kRotMaxPairs = 128;
constexpr int kRotMaxAxes = 4;

struct RotArgs {
    const void* x[2];
    void* y[2];
    long long sb[2], sn[2], sh[2];      // strides of x (elements); y is contiguous [B, N, H, D]
    int H[2];
    const void* pos;                    // [B or 1, N, axes]
    long long psb, psn;                 // strides of pos (elements), last axis contiguous
    int pos_type;                       // 0 int32, 1 int64, 2 fp32
    int B, N, D, R, items;              // items: work items per token
    long long total;                    // B * N * items
    int heads_per_group;
    float sign;
    double turns[kRotMaxPairs];         // f_j / (2 pi)
    unsigned char axis[kRotMaxPairs];
};

// the fused multiply-adds are written out: the 16-byte and the single-element form give the same bits
template <typename T, int E> struct RotVec { typedef T type __attribute__((ext_vector_type(E))); };

// E: elements per access (16 bytes, or 1). HALF: pair (j, j + R/2), otherwise (2 j, 2 j + 1).
// items of a token: HALF: (R/2) / E rotating (two accesses each) | adjacent: R / EA rotating (one access of EA = max(E, 2)); then (D - R) / E passing
template <typename T, int E, bool HALF>
__global__ __launch_bounds__(256) void rotary_axes_kernel(RotArgs a) {
    constexpr int EA = HALF ? E : (E < 2 ? 2 : E);              // elements of a rotating access
    constexpr int NP = HALF ? E : EA / 2;                       // pairs of a rotating item
    typedef typename RotVec<T, E>::type VE;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.total) return;
    const long long tok = id / a.items;
    const int c = (int)(id - tok * a.items);
    const int b = (int)(tok / a.N), n = (int)(tok - (long long)b * a.N);
    const int rot_items = HALF ? (a.R >> 1) / E : a.R / EA;
    const int heads = a.H[0] + a.H[1];
    const int h0 = blockIdx.y * a.heads_per_group;
    const int h1 = h0 + a.heads_per_group < heads ? h0 + a.heads_per_group : heads;

    if (c >= rot_items) {                                       // passing channels
        const int e0 = a.R + (c - rot_items) * E;
        for (int hh = h0; hh < h1; ++hh) {
            const int s = hh >= a.H[0];
            const int h = s ? hh - a.H[0] : hh;
            const T* src = (const T*)a.x[s] + b * a.sb[s] + n * a.sn[s] + h * a.sh[s] + e0;
            T* dst = (T*)a.y[s] + ((tok * a.H[s]) + h) * a.D + e0;
            if constexpr (E == 1) *dst = *src;
            else *reinterpret_cast<VE*>(dst) = *reinterpret_cast<const VE*>(src);
        }
        return;
    }

    const long long prow = b * a.psb + n * a.psn;
    float cs[NP], sn[NP];
    const int j0 = c * NP;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int ax = a.axis[j0 + i];
        double p;
        if (a.pos_type == 0) p = (double)((const int*)a.pos)[prow + ax];
        else if (a.pos_type == 1) p = (double)((const long long*)a.pos)[prow + ax];
        else p = (double)((const float*)a.pos)[prow + ax];
        const double t4 = 4.0 * (p * a.turns[j0 + i]);          // quarter turns
        const double q = rint(t4);
        float s, co;
        sincospif(0.5f * (float)(t4 - q), &s, &co);
        const int k = (int)(q - 4.0 * floor(0.25 * q));         // whole quarters, 0 .. 3
        const float cc = (k & 1) ? s : co, ss = (k & 1) ? co : s;
        cs[i] = (k == 1 || k == 2) ? -cc : cc;                  // turn by k quarters: (c, s) -> (-s, c) -> (-c, -s) -> (s, -c)
        sn[i] = a.sign * (k >= 2 ? -ss : ss);
    }

    auto walk = [&](int s, int ha, int hb) {
        const T* src = (const T*)a.x[s] + b * a.sb[s] + n * a.sn[s];
        T* dst = (T*)a.y[s] + (tok * a.H[s]) * a.D;
#pragma unroll 4
        for (int h = ha; h < hb; ++h) {
            const T* p = src + h * a.sh[s];
            T* o = dst + (long long)h * a.D;
            if constexpr (HALF) {
                const int e0 = c * E, e1 = e0 + (a.R >> 1);
                if constexpr (E == 1) {
                    const float u = (float)p[e0], v = (float)p[e1];
                    o[e0] = (T)fmaf(u, cs[0], -(v * sn[0]));
                    o[e1] = (T)fmaf(v, cs[0], u * sn[0]);
                } else {
                    const VE u = *reinterpret_cast<const VE*>(p + e0), v = *reinterpret_cast<const VE*>(p + e1);
                    VE yu, yv;
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        yu[i] = (T)fmaf((float)u[i], cs[i], -((float)v[i] * sn[i]));
                        yv[i] = (T)fmaf((float)v[i], cs[i], (float)u[i] * sn[i]);
                    }
                    *reinterpret_cast<VE*>(o + e0) = yu;
                    *reinterpret_cast<VE*>(o + e1) = yv;
                }
            } else {
                const int e0 = c * EA;
                if constexpr (E == 1) {
                    const float u = (float)p[e0], v = (float)p[e0 + 1];
                    o[e0] = (T)fmaf(u, cs[0], -(v * sn[0]));
                    o[e0 + 1] = (T)fmaf(v, cs[0], u * sn[0]);
                } else {
                    const VE x = *reinterpret_cast<const VE*>(p + e0);
                    VE y;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const float u = (float)x[2 * i], v = (float)x[2 * i + 1];
                        y[2 * i] = (T)fmaf(u, cs[i], -(v * sn[i]));
                        y[2 * i + 1] = (T)fmaf(v, cs[i], u * sn[i]);
                    }
                    *reinterpret_cast<VE*>(o + e0) = y;
                }
            }
        }
    };
    const int m0 = h1 < a.H[0] ? h1 : a.H[0];
    if (h0 < m0) walk(0, h0, m0);
    const int k0 = h0 > a.H[0] ? h0 - a.H[0] : 0;
    if (h1 > a.H[0]) walk(1, k0, h1 - a.H[0]);
}

template <typename T, int E, bool HALF>
int rotary_launch(RotArgs& a, void* stream) {
    const int rot = HALF ? (a.R >> 1) / E : a.R / (E < 2 ? 2 : E);
    a.items = rot + (a.D - a.R) / E;
    a.total = (long long)a.B * a.N * a.items;
    const long long wgs = (a.total + 255) / 256;
    if (wgs > 0x7fffffffLL) return SVPS_ERR_BAD_SHAPE;
    // enough work items for 8 waves per SIMD's worth of loads in flight (4 workgroups per CU): below that the heads are dealt out
    const int heads = a.H[0] + a.H[1];
    const long long want = 4LL * svps_num_cus();
    long long groups = wgs >= want ? 1 : (want + wgs - 1) / wgs;
    if (groups > heads) groups = heads;
    a.heads_per_group = (heads + (int)groups - 1) / (int)groups;
    const int gy = (heads + a.heads_per_group - 1) / a.heads_per_group;
    hipLaunchKernelGGL((rotary_axes_kernel<T, E, HALF>), dim3((unsigned)wgs, gy), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return (int)hipGetLastError();
}

template <typename T>
int rotary_dispatch(RotArgs& a, int pairing, void* stream) {
    constexpr int E = 16 / sizeof(T);
    // 16-byte accesses where every row of both tensors starts on 16 bytes and no access straddles the end of a section
    bool vec = (pairing == 0 ? (a.R >> 1) % E == 0 : a.R % E == 0) && a.D % E == 0;
    for (int s = 0; s < 2; ++s)
        if (a.H[s]) vec = vec && !((uintptr_t)a.x[s] & 15) && !((uintptr_t)a.y[s] & 15) && a.sb[s] % E == 0 && a.sn[s] % E == 0 && a.sh[s] % E == 0;
    if (pairing == 0) return vec ? rotary_launch<T, E, true>(a, stream) : rotary_launch<T, 1, true>(a, stream);
    return vec ? rotary_launch<T, E, false>(a, stream) : rotary_launch<T, 1, false>(a, stream);
}

}  // namespace svps

extern "C" int svps_rotary_axes(const void* x, const long long* sx, void* y, int H, const void* x2, const long long* sx2, void* y2, int H2,
                                const void* pos, long long pos_sb, long long pos_sn, int pos_type, int axes, const int* split,
                                const double* turns, int pairing, int inverse, int dtype, int B, int N, int D, void* stream) {
    using namespace svps;
    if (!x || !sx || !y || !pos || !split || !turns || (H2 > 0 && (!x2 || !sx2 || !y2))) return SVPS_ERR_BAD_ARG;
    if (pos_type < 0 || pos_type > 2 || pairing < 0 || pairing > 1 || dtype < 0 || dtype > 2) return SVPS_ERR_BAD_ARG;
    if (B <= 0 || N <= 0 || H <= 0 || H2 < 0 || D <= 0 || D > 4096 || axes < 1 || axes > kRotMaxAxes) return SVPS_ERR_BAD_SHAPE;
    if (H > 65535 - H2) return SVPS_ERR_BAD_SHAPE;
    RotArgs a = {};
    int pairs = 0;
    for (int i = 0; i < axes; ++i) {
        if (split[i] < 2 || (split[i] & 1) || split[i] > 2 * kRotMaxPairs || pairs + split[i] / 2 > kRotMaxPairs) return SVPS_ERR_BAD_SHAPE;
        for (int j = 0; j < split[i] / 2; ++j) a.axis[pairs++] = (unsigned char)i;
    }
    if (2 * pairs > D) return SVPS_ERR_BAD_SHAPE;
    for (int j = 0; j < pairs; ++j) a.turns[j] = turns[j];
    a.x[0] = x; a.y[0] = y; a.H[0] = H; a.sb[0] = sx[0]; a.sn[0] = sx[1]; a.sh[0] = sx[2];
    if (H2 > 0) { a.x[1] = x2; a.y[1] = y2; a.H[1] = H2; a.sb[1] = sx2[0]; a.sn[1] = sx2[1]; a.sh[1] = sx2[2]; }
    a.pos = pos; a.psb = pos_sb; a.psn = pos_sn; a.pos_type = pos_type;
    a.B = B; a.N = N; a.D = D; a.R = 2 * pairs;
    a.sign = inverse ? -1.f : 1.f;
    if (dtype == SVPS_DTYPE_BF16) return rotary_dispatch<__bf16>(a, pairing, stream);
    if (dtype == SVPS_DTYPE_F16) return rotary_dispatch<_Float16>(a, pairing, stream);
    return rotary_dispatch<float>(a, pairing, stream);
}
