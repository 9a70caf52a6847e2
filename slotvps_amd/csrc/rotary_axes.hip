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
// Bound: bandwidth (each value read once, written once; 6 operations per pair). A workgroup takes a few tokens: the cosines and sines of
// their pairs once, into LDS, then all heads of both tensors as a stream of 16-byte pieces, consecutive lanes on consecutive pieces (a lane
// per pair of pieces with the heads in a loop reads the same bytes in 96-byte shreds: 40960 tokens, 20 heads of 128: 143 us against 90 us = 4.7 TB/s). The
// other half of a pair is a second read of a line that the wave has just asked for. Few tokens: the heads are dealt over grid.y. fp32: 163 us =
// 5.1 TB/s. Rows that are not aligned and sections that end inside a piece go by single elements, one in flight: at R = 40 302 us = 1.4 TB/s.
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
    int B, N, D, R, tokens_per_wg, heads_per_group;
    float sign;
    double turns[kRotMaxPairs];         // f_j / (2 pi)
    unsigned char axis[kRotMaxPairs];
};

// the fused multiply-adds are written out: the 16-byte and the single-element form give the same bits
template <typename T, int E> struct RotVec { typedef T type __attribute__((ext_vector_type(E))); };
template <typename T> struct RotVec<T, 1> { typedef T type; };

constexpr int kRotTable = 1024;         // pairs of a workgroup's tokens

// E: elements of a piece (16 bytes, or 1 where rows are not aligned or sections end inside a piece). HALF: pair (j, j + R/2), else (2 j, 2 j + 1)
template <typename T, int E, bool HALF>
__global__ __launch_bounds__(256) void rotary_axes_kernel(RotArgs a) {
    constexpr int U = E == 1 ? 1 : 4;                            // pieces in flight
    constexpr int NP = HALF ? E : (E + 1) / 2;                  // pairs of a piece
    typedef typename RotVec<T, E>::type VE;
    __shared__ float2 tab[kRotTable];
    const int pairs = a.R >> 1, tid = threadIdx.x;
    const long long tokens = (long long)a.B * a.N, t0 = (long long)blockIdx.x * a.tokens_per_wg;
    const int nt = (int)(tokens - t0 < a.tokens_per_wg ? tokens - t0 : a.tokens_per_wg);
    for (int i = tid; i < nt * pairs; i += 256) {
        const int k = i / pairs, j = i - k * pairs;
        const long long tok = t0 + k, b = tok / a.N, at = b * a.psb + (tok - b * a.N) * a.psn + a.axis[j];
        double p;
        if (a.pos_type == 0) p = (double)((const int*)a.pos)[at];
        else if (a.pos_type == 1) p = (double)((const long long*)a.pos)[at];
        else p = (double)((const float*)a.pos)[at];
        const double t4 = 4.0 * (p * a.turns[j]);               // quarter turns
        const double q = rint(t4);
        float s, co;
        sincospif(0.5f * (float)(t4 - q), &s, &co);
        const int quarter = (int)(q - 4.0 * floor(0.25 * q));   // whole quarters, 0 .. 3
        const float cc = (quarter & 1) ? s : co, ss = (quarter & 1) ? co : s;
        // turn by whole quarters: (c, s) -> (-s, c) -> (-c, -s) -> (s, -c)
        tab[i] = make_float2(quarter == 1 || quarter == 2 ? -cc : cc, a.sign * (quarter >= 2 ? -ss : ss));
    }
    __syncthreads();

    const int heads = a.H[0] + a.H[1];
    const int h0 = blockIdx.y * a.heads_per_group;
    const int h1 = h0 + a.heads_per_group < heads ? h0 + a.heads_per_group : heads;
    const int per_head = a.D / E, half = a.R >> 1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int ha = s ? (h0 > a.H[0] ? h0 - a.H[0] : 0) : h0, hb = s ? h1 - a.H[0] : (h1 < a.H[0] ? h1 : a.H[0]);
        if (ha >= hb) continue;
        const int nh = hb - ha;
        // piece (token k, head h, piece c) of this thread, and the step of 256 pieces as such digits
        int c = tid % per_head, h = (tid / per_head) % nh, k = tid / per_head / nh;
        const int dc = 256 % per_head, dh = (256 / per_head) % nh, dk = 256 / per_head / nh;
        while (k < nt) {
            VE own[U], other[U];
            int pc[U], pk[U];
            T* dst[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                pk[u] = k;
                pc[u] = c;
                if (k < nt) {
                    const long long tok = t0 + k, b = tok / a.N;
                    const T* src = (const T*)a.x[s] + b * a.sb[s] + (tok - b * a.N) * a.sn[s] + (long long)(ha + h) * a.sh[s];
                    dst[u] = (T*)a.y[s] + (tok * a.H[s] + ha + h) * a.D + c * E;
                    const int e = c * E;
                    own[u] = *reinterpret_cast<const VE*>(src + e);
                    if (HALF) other[u] = *reinterpret_cast<const VE*>(src + (e < half ? e + half : e < a.R ? e - half : e));
                    else if (E == 1) other[u] = *reinterpret_cast<const VE*>(src + (e < a.R ? e ^ 1 : e));
                }
                c += dc;
                h += dh;
                k += dk;
                if (c >= per_head) { c -= per_head; ++h; }
                if (h >= nh) { h -= nh; ++k; }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (pk[u] >= nt) break;
                const int e = pc[u] * E;
                VE y = own[u];
                if (e < a.R) {
                    const bool second = HALF ? e >= half : false;
                    const float2* t = tab + pk[u] * pairs + (HALF ? (second ? e - half : e) : e >> 1);
                    if constexpr (HALF || E == 1) {
#pragma unroll
                        for (int i = 0; i < E; ++i) {
                            const float co = t[i].x, si = t[i].y;
                            float x, z;
                            if constexpr (E == 1) { x = (float)own[u]; z = (float)other[u]; }
                            else { x = (float)own[u][i]; z = (float)other[u][i]; }
                            const bool hi = HALF ? second : (e & 1);
                            const float v = hi ? fmaf(x, co, z * si) : fmaf(x, co, -(z * si));
                            if constexpr (E == 1) y = (T)v;
                            else y[i] = (T)v;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            const float u0 = (float)own[u][2 * i], v0 = (float)own[u][2 * i + 1];
                            y[2 * i] = (T)fmaf(u0, t[i].x, -(v0 * t[i].y));
                            y[2 * i + 1] = (T)fmaf(v0, t[i].x, u0 * t[i].y);
                        }
                    }
                }
                *reinterpret_cast<VE*>(dst[u]) = y;
            }
        }
    }
}

template <typename T, int E, bool HALF>
int rotary_launch(RotArgs& a, void* stream) {
    const int heads = a.H[0] + a.H[1], cus = svps_num_cus();
    const long long tokens = (long long)a.B * a.N;
    // tokens of a workgroup: eight pieces per thread, as far as the table holds them, fewer where that leaves a CU without four workgroups;
    // one each and still fewer: the heads are dealt out
    long long per = kRotTable / (a.R >> 1);
    const long long pieces = (long long)heads * (a.D / E), many = (2048 + pieces - 1) / pieces;
    if (per > many) per = many;
    if (per > tokens / (4 * cus)) per = tokens / (4 * cus);
    if (per < 1) per = 1;
    const long long wgs = (tokens + per - 1) / per;
    if (wgs > 0x7fffffffLL) return SVPS_ERR_BAD_SHAPE;
    long long groups = wgs >= 4 * cus ? 1 : (4 * cus + wgs - 1) / wgs;
    const long long least = (256 * E + a.D - 1) / a.D;           // heads that give every thread a piece
    if (groups > (heads + least - 1) / least) groups = (heads + least - 1) / least;
    a.tokens_per_wg = (int)per;
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
