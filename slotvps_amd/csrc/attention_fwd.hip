// Attention forward (attention.h has the mathematics and the layouts): one pass over the keys with the running maximum and sum of the
// softmax, fp32 throughout; probabilities are rounded to 16 bits once, as the operand of the product with the values.
//
// Workgroup = NW waves x 32 packed rows of one (batch entry, key head) pair; key / value tiles of KT rows in LDS, double-buffered by
// LDS-DMA (the next tile flies under this one's products), one barrier per tile. Few rows: the key range is split over `splits`
// workgroups that leave unnormalised sums with their maximum, joined by att_combine_kernel.
#include "attention.h"
#include "../../include/slotvps_hip.h"

namespace svps {

template <typename T, int DP, int NW, int KT>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void attention_fwd_kernel(AttArgs a) {
    typedef typename AttVec<T>::v8 v8;
    constexpr int KS = DP / 16, DB = DP / 32, KB = KT / 32, TILE = KT * DP * 2;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = a.B * a.Hk;
    const int id = blockIdx.x;
    const int rest = id / pairs;
    const int pair = att_pair(id, rest, pairs);
    const int t = a.tiles - 1 - rest % a.tiles;                    // late rows see the most keys in causal order: longest first
    const int split = rest / a.tiles;
    const int b = pair / a.Hk, hk = pair - b * a.Hk;
    const int qlen = att_qlen(a, b), klen = att_klen(a, b);

    const int row0 = (t * NW + w) * 32;                            // the wave's rows
    const int row = row0 + r;
    const int n = att_div_g(a, row);
    const int head = hk * a.G + (row - n * a.G);
    const bool have = n < qlen;
    const long long orow = ((long long)b * a.N + n) * a.H + head;  // row of out / of the partial sums (n < N only)

    const int wg0 = att_div_g(a, t * NW * 32);
    if (wg0 >= qlen) {                                             // nothing valid in the workgroup: zeros, and leave
        if (n < a.N && split == 0) {
            T* o = (T*)a.out + orow * a.D;
            for (int d = 8 * h; d < a.D; d += 16) *reinterpret_cast<u32x4*>(o + d) = u32x4{0, 0, 0, 0};
            if (a.lse && h == 0) a.lse[((long long)b * a.H + head) * a.N + n] = -INFINITY;
        }
        if (a.splits > 1 && n < a.N && h == 0) {
            float* ml = a.part + (long long)a.splits * a.B * a.N * a.H * a.D + (split * ((long long)a.B * a.N * a.H) + orow) * 2;
            ml[0] = 0.f;
            ml[1] = 0.f;
        }
        return;
    }
    int wg1 = att_div_g(a, t * NW * 32 + NW * 32 - 1);
    wg1 = wg1 < qlen ? wg1 : qlen - 1;
    int lo_wg, hi_wg, lo, hi, tmp;
    att_range(a, wg0, qlen, klen, lo_wg, tmp);
    att_range(a, wg1, qlen, klen, tmp, hi_wg);
    att_range(a, have ? n : qlen - 1, qlen, klen, lo, hi);
    // the wave's bounds: [lo_min, hi_max) is visited, [lo_max, hi_min) needs no comparison
    const int wn0 = att_div_g(a, row0);
    int wn1 = att_div_g(a, row0 + 31);
    wn1 = wn1 < qlen ? wn1 : qlen - 1;
    const bool wave_on = wn0 < qlen;
    int lo_min, hi_min, lo_max, hi_max;
    att_range(a, wave_on ? wn0 : qlen - 1, qlen, klen, lo_min, hi_min);
    att_range(a, wn1, qlen, klen, lo_max, hi_max);

    int tb = lo_wg / KT, te = hi_wg > lo_wg ? (hi_wg + KT - 1) / KT : lo_wg / KT;
    if (a.splits > 1) {
        const int per = (te - tb + a.splits - 1) / a.splits;
        tb += split * per;
        te = tb + per < te ? tb + per : te;
    }

    v8 qf[KS];
    {
        const T* qp = (const T*)a.q + b * a.sqb + n * a.sqn + head * a.sqh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 16 * ks + 8 * h;
            u32x4 x = {0, 0, 0, 0};
            if (have && d < a.D) x = *reinterpret_cast<const u32x4*>(qp + d);
            qf[ks] = __builtin_bit_cast(v8, x);
        }
    }

    AttTile<DP, KT, NW, kAttK> tk;
    AttTile<DP, KT, NW, kAttV> tv;
    tk.init((const T*)a.k + b * a.skb + hk * a.skh, a, w, lane);
    tv.init((const T*)a.v + b * a.svb + hk * a.svh, a, w, lane);
    auto stage = [&](int tile, int buf) __attribute__((always_inline)) {
        char* lk = smem + buf * 2 * TILE;
        tk.stage(tile, klen, lk, w, lane);
        tv.stage(tile, klen, lk + TILE, w, lane);
    };

    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
    const float c = a.scale * kLog2e;
    AttLane<DP> at(lane);
    float mc = kAttFloor, l = 0.f;                                 // reference point of the exponentials (base 2) and their sum (this lane half's keys)

    if (tb < te) stage(tb, 0);
    for (int tile = tb; tile < te; ++tile) {
        const int buf = (tile - tb) & 1;
        wait_vm<0>();
        wg_barrier();                                              // the tile is here; nobody reads the other buffer any more
        if (tile + 1 < te) stage(tile + 1, buf ^ 1);
        const int k0 = tile * KT;
        if (!wave_on || k0 >= hi_max || k0 + KT <= lo_min) continue;
        const char* lk = smem + buf * 2 * TILE;
        const char* lv = lk + TILE;
        at.pin();
        float p[KB * 16];
        float mt = -INFINITY;
        const bool whole = k0 >= lo_max && k0 + KT <= hi_min;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = mfma16(att_row_frag<T, DP>(lk, at, 32 * kb, ks), qf[ks], s);
#pragma unroll
            for (int i = 0; i < 16; ++i) p[16 * kb + i] = s[i];
        }
        if (!whole) {
            asm volatile("");                                      // a branch, not 32 selects in every tile
#pragma unroll
            for (int i = 0; i < KB * 16; ++i) {
                const int key = k0 + 32 * (i >> 4) + acc_row(i & 15, h);
                if (key < lo || key >= hi) p[i] = -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < KB * 16; ++i) mt = fmaxf(mt, p[i]);
        // The reference point of the exponentials moves only when a row's maximum has outgrown it by a factor of 2^8: until then the sums
        // stay within 2^8 of their scale, and the rescaling (every accumulator of the wave) is skipped.
        if (__any(mt * c > mc + 8.f)) {
            const float mn = fmaxf(mc, wave_half_xor_max(mt) * c);     // a row's keys are in both lane halves: one point for both
            const float alpha = __builtin_amdgcn_exp2f(mc - mn);
            mc = mn;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < KB * 16; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], c, -mc));
            l += p[i];                                             // before its rounding: the backward pass divides by this sum
        }
#pragma unroll
        for (int ks = 0; ks < KT / 16; ++ks) {
            const v8 pf = att_pack<T>(p + 8 * ks);
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = mfma16(att_col_frag<T, DP>(lv, at, 16 * ks, db), pf, acc[db]);
        }
    }

    l = wave_half_xor_sum(l);
    if (n >= a.N) return;
    if (a.splits > 1) {
        const long long rows = (long long)a.B * a.N * a.H;
        float* po = a.part + (split * rows + orow) * a.D;
#pragma unroll
        for (int db = 0; db < DB; ++db) att_store_block_f32(po, 32 * db, h, a.D, acc[db]);
        if (h == 0) {
            float* ml = a.part + (long long)a.splits * rows * a.D + (split * rows + orow) * 2;
            ml[0] = mc;
            ml[1] = have ? l : 0.f;
        }
        return;
    }
    const bool some = have && l > 0.f;
    T* o = (T*)a.out + orow * a.D;
    if (some) {
        const float inv = 1.f / l;
#pragma unroll
        for (int db = 0; db < DB; ++db) att_store_block<T>(o, 32 * db, h, a.D, acc[db], inv);
    } else {                                                       // no visible key, or a row behind qlen
        for (int d = 8 * h; d < a.D; d += 16) *reinterpret_cast<u32x4*>(o + d) = u32x4{0, 0, 0, 0};
    }
    if (a.lse && h == 0) a.lse[((long long)b * a.H + head) * a.N + n] = some ? (mc + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

// joins the splits of a row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s. One workgroup per row: every lane of a wave holds the
// weight of one split (splits <= 64), thread (g, c) adds splits g, g + 8, .. of channels 4 c .. 4 c + 3, the eight sums meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void attention_combine_kernel(AttArgs a) {
    __shared__ float red[8][128];
    __shared__ float wt[64];
    const long long rows = (long long)a.B * a.N * a.H;
    const long long row = blockIdx.x;
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 5, c = (threadIdx.x & 31) * 4;
    const float* ml = a.part + (long long)a.splits * rows * a.D;
    float ms = -INFINITY, ls = 0.f;
    if (lane < a.splits) {
        const float2 x = *reinterpret_cast<const float2*>(ml + (lane * rows + row) * 2);
        ls = x.y;
        ms = ls > 0.f ? x.x : -INFINITY;
    }
    float m = ms;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float f = ls > 0.f ? exp2f(ms - m) : 0.f;
    float l = f * ls;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
    if (threadIdx.x < 64) wt[lane] = f;
    __syncthreads();
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < a.D) {
#pragma unroll 4
        for (int k = g; k < a.splits; k += 8) {
            const float w = wt[k];
            if (w > 0.f) {                                         // a split without keys left its sums unwritten
                const f32x4 o = *reinterpret_cast<const f32x4*>(a.part + (k * rows + row) * a.D + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += w * o[j];
            }
        }
    }
    *reinterpret_cast<f32x4*>(&red[g][c]) = s;
    __syncthreads();
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (threadIdx.x < a.D) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += red[k][threadIdx.x];
        ((T*)a.out)[row * a.D + threadIdx.x] = (T)(t * inv);
    }
    if (a.lse && threadIdx.x == 0) {
        const int h = (int)(row % a.H);
        const long long bn = row / a.H;
        const int n = (int)(bn % a.N);
        const long long b = bn / a.N;
        a.lse[(b * a.H + h) * a.N + n] = l > 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    }
}

struct AttPlan { int nw, kt, tiles, splits; };

static AttPlan attention_plan(int B, int N, int M, int H, int Hk) {
    const long long rows = (long long)N * (H / Hk), pairs = (long long)B * Hk;
    AttPlan p;
    p.nw = rows <= 32 ? 1 : 4;
    p.kt = p.nw == 1 ? 32 : 64;
    p.tiles = (int)((rows + 32 * p.nw - 1) / (32 * p.nw));
    const long long wgs = pairs * p.tiles, want = (p.nw == 1 ? 4LL : 2LL) * svps_num_cus();
    const long long key_tiles = (M + p.kt - 1) / p.kt;
    long long s = wgs * 2 > want ? 1 : want / wgs;
    if (s > key_tiles / 4) s = key_tiles / 4;
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

template <typename T, int DP, int NW, int KT>
static int attention_launch(const AttArgs& a, hipStream_t stream) {
    static SvpsLdsAttr attr;
    constexpr int LDS = 4 * KT * DP * 2;
    const hipError_t e = attr.ensure((const void*)attention_fwd_kernel<T, DP, NW, KT>, LDS);
    if (e != hipSuccess) return (int)e;
    const unsigned grid = (unsigned)((long long)a.B * a.Hk * a.tiles * a.splits);
    hipLaunchKernelGGL((attention_fwd_kernel<T, DP, NW, KT>), dim3(grid), dim3(64 * NW), LDS, stream, a);
    return (int)hipGetLastError();
}

template <typename T>
static int attention_dispatch(const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    int rc;
    if (p.nw == 1) rc = a.D <= 32 ? attention_launch<T, 32, 1, 32>(a, stream) : a.D <= 64 ? attention_launch<T, 64, 1, 32>(a, stream) : attention_launch<T, 128, 1, 32>(a, stream);
    else rc = a.D <= 32 ? attention_launch<T, 32, 4, 64>(a, stream) : a.D <= 64 ? attention_launch<T, 64, 4, 64>(a, stream) : attention_launch<T, 128, 4, 64>(a, stream);
    if (rc || a.splits == 1) return rc;
    const long long rows = (long long)a.B * a.N * a.H;
    hipLaunchKernelGGL(attention_combine_kernel<T>, dim3((unsigned)rows), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int attention_check(const void* const* ptrs, int np, const long long* const* strides, int ns, int B, int N, int M, int H, int Hk, int D,
                    int frame, int window, float scale, int dtype) {
    for (int i = 0; i < np; ++i) {
        if (!ptrs[i]) return SVPS_ERR_BAD_ARG;
        if ((uintptr_t)ptrs[i] & 15) return SVPS_ERR_BAD_ARG;
    }
    for (int i = 0; i < ns; ++i) {
        if (!strides[i]) return SVPS_ERR_BAD_ARG;
        for (int j = 0; j < 3; ++j) if (strides[i][j] & 7) return SVPS_ERR_BAD_ARG;
    }
    if (dtype != SVPS_DTYPE_BF16 && dtype != SVPS_DTYPE_F16) return SVPS_ERR_BAD_ARG;
    if (!(scale > 0.f) || scale > 1e30f || frame < 0 || window < 0 || (window > 0 && frame == 0)) return SVPS_ERR_BAD_ARG;
    if (B <= 0 || N <= 0 || M <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || D > 128 || D % 8) return SVPS_ERR_BAD_SHAPE;
    const int big = 1 << 30;
    if (M > big || frame > big || (long long)N * (H / Hk) > big) return SVPS_ERR_BAD_SHAPE;
    if ((long long)B * Hk * (((long long)N * (H / Hk) + 31) / 32 + (M + 31) / 32) > big) return SVPS_ERR_BAD_SHAPE;
    return 0;
}

}  // namespace svps

extern "C" size_t svps_attention_workspace_bytes(int B, int N, int M, int H, int Hk, int D) {
    if (B <= 0 || N <= 0 || M <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0) return 0;
    const svps::AttPlan p = svps::attention_plan(B, N, M, H, Hk);
    return p.splits > 1 ? (size_t)p.splits * B * N * H * (D + 2) * sizeof(float) : 0;
}

extern "C" int svps_attention_fwd(const void* q, const long long* sq, const void* k, const long long* sk, const void* v, const long long* sv,
                                  void* out, float* lse, const int* qlens, const int* klens, void* workspace, size_t workspace_bytes,
                                  int B, int N, int M, int H, int Hk, int D, int frame, int window, float scale, int dtype, void* stream) {
    using namespace svps;
    const void* ptrs[] = {q, k, v, out};
    const long long* st[] = {sq, sk, sv};
    const int rc = attention_check(ptrs, 4, st, 3, B, N, M, H, Hk, D, frame, window, scale, dtype);
    if (rc) return rc;
    const AttPlan p = attention_plan(B, N, M, H, Hk);
    const size_t need = svps_attention_workspace_bytes(B, N, M, H, Hk, D);
    if (need && (!workspace || workspace_bytes < need)) return SVPS_ERR_WORKSPACE;
    AttArgs a = {};
    a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse; a.qlens = qlens; a.klens = klens;
    a.sqb = sq[0]; a.sqn = sq[1]; a.sqh = sq[2]; a.skb = sk[0]; a.skn = sk[1]; a.skh = sk[2]; a.svb = sv[0]; a.svn = sv[1]; a.svh = sv[2];
    a.part = (float*)workspace;
    a.B = B; a.N = N; a.M = M; a.H = H; a.Hk = Hk; a.G = H / Hk; a.D = D; a.frame = frame; a.window = window;
    a.splits = p.splits; a.tiles = p.tiles; a.scale = scale;
    a.gmagic = a.G > 1 ? (unsigned)(0x100000000ULL / a.G) + 1 : 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SVPS_DTYPE_BF16 ? attention_dispatch<__bf16>(a, p, s) : attention_dispatch<_Float16>(a, p, s);
}
