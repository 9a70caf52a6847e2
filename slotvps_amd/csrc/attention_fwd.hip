// Attention forward (attention.h has the mathematics and the layouts): one pass over the keys with the running maximum and sum of the
// softmax, fp32 throughout; probabilities are rounded to 16 bits once, as the operand of the product with the values.
//
// Workgroup = NW waves x 32 packed rows of one (batch entry, key head) pair; key / value tiles of KT rows in LDS, double-buffered by
// LDS-DMA (the next tile flies under this one's products), one barrier per tile. Few rows: the key range is split over `splits`
// workgroups that leave unnormalised sums with their maximum, joined by attention_combine_kernel.
//
// Bound: the matrix products (4 D flop per visible pair) and the softmax beside them - at heads of 128 about 40 vector instructions and 16
// exponentials for 8 products of 32 x 32 x 16, at heads of 32 as many for 4. Measured in bf16: 4 x 4096 tokens, 16 heads of 128 528 us =
// 1041 TFLOP/s, causal 294 us = 934 TFLOP/s; 10240 tokens, 8 heads of 64 271 us = 792, of 32 204 us = 526 TFLOP/s. A single query over a long
// memory is bound by its bytes: 5 x up to 16383 keys (126 MB in all), 4 heads of 128 23.4 us = 5.4 TB/s. Head sizes between are multiplied as
// the next of 32, 64 and 128 and staged by per-lane addresses: 4 x 4096 tokens, 16 heads of 40 311 us, of 72 546 us, of 96 560 us.
//
// Scores in base 2 (scale log2 e q k) hold to 2^30 in magnitude: a score is compared with the row's reference point in one fused multiply-add,
// whose exact result is up to the rounding of that point away from 0 - beyond 2^31 more than exp2 can take, the row becomes NaN.
#include "attention.h"
#include "../../include/slotvps_hip.h"

namespace svps {

template <typename T, int DP, int NW, int KT, int RB>
// DP = 128: LDS admits two waves per SIMD; told so, the compiler uses their registers to read fragments ahead (4097 causal tokens: 148 -> 137 us)
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP == 128 || NW == 1 ? 2 : 4, DP == 128 ? 2 : 8))) void attention_fwd_kernel(AttArgs a) {
    typedef typename AttVec<T>::v8 v8;
    constexpr int KS = DP / 16, DB = DP / 32, TILE = KT * DP * 2, ROWS = 32 * RB;
    constexpr int KB = KT == 32 || (RB == 2 && DP == 128) ? 1 : 2;   // blocks of 32 keys whose scores are held at a time
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
    const int row0 = (t * NW + w) * ROWS;                          // the wave's first row; a lane owns rows row0 + 32 i + r
    const int wg0 = att_div_g(a, t * NW * ROWS);

    v8 qf[RB][KS];
    int tb = 0, te = 0, lo_min = 0, hi_min = 0, lo_max = 0, hi_max = 0;
    const int wn0 = att_div_g(a, row0);
    const bool wave_on = wn0 < qlen;
    if (wg0 < qlen) {
        int wg1 = att_div_g(a, t * NW * ROWS + NW * ROWS - 1);
        wg1 = wg1 < qlen ? wg1 : qlen - 1;
        int lo_wg, hi_wg, tmp;
        att_range(a, wg0, qlen, klen, lo_wg, tmp);
        att_range(a, wg1, qlen, klen, tmp, hi_wg);
        // the wave's bounds: [lo_min, hi_max) is visited, [lo_max, hi_min) needs no comparison
        int wn1 = att_div_g(a, row0 + ROWS - 1);
        wn1 = wn1 < qlen ? wn1 : qlen - 1;
        att_range(a, wave_on ? wn0 : qlen - 1, qlen, klen, lo_min, hi_min);
        att_range(a, wn1, qlen, klen, lo_max, hi_max);
        tb = lo_wg / KT;
        te = hi_wg > lo_wg ? (hi_wg + KT - 1) / KT : tb;
        if (a.splits > 1) {
            const int per = (te - tb + a.splits - 1) / a.splits;
            tb += split * per;
            te = tb + per < te ? tb + per : te;
        }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int row = row0 + 32 * i + r, n = att_div_g(a, row), head = hk * a.G + (row - n * a.G);
        const bool have = n < qlen;
        const T* qp = (const T*)a.q + b * a.sqb + n * a.sqn + head * a.sqh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 16 * ks + 8 * h;
            u32x4 x = {0, 0, 0, 0};
            if (have && d < a.D) x = *reinterpret_cast<const u32x4*>(qp + d);
            qf[i][ks] = __builtin_bit_cast(v8, x);
        }
    }

    constexpr bool HOLD = RB == 1;
    AttTile<DP, KT, NW, kAttK, HOLD> tk;
    AttTile<DP, KT, NW, kAttV, HOLD> tv;
    tk.init((const T*)a.k + b * a.skb + hk * a.skh, a, w, lane);
    tv.init((const T*)a.v + b * a.svb + hk * a.svh, a, w, lane);
    f32x16 acc[RB][DB];
    float mc[RB], l[RB];                                           // reference point of the exponentials (base 2) and their sum (this lane half's keys)
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        mc[i] = kAttFloor;
        l[i] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][db][e] = 0.f;
    }
    const float c = a.scale * kLog2e;
    AttLane<DP> at(lane);

    auto stage = [&](int tile, int buf) __attribute__((always_inline)) {
        char* lk = smem + buf * 2 * TILE;
        tk.stage(tile, klen, lk, w);
        tv.stage(tile, klen, lk + TILE, w);
    };
    if (tb < te) stage(tb, 0);
    for (int tile = tb; tile < te; ++tile) {
        const int buf = (tile - tb) & 1;
        wait_vm<0>();
        wg_barrier();                                              // the tile is here; nobody reads the other buffer any more
        const char* lk = smem + buf * 2 * TILE;
        const char* lv = lk + TILE;
        bool asked = tile + 1 >= te;                               // the next tile: asked for behind the first products
#pragma unroll 1
        for (int sub = 0; sub < KT / (32 * KB); ++sub) {
            const int k0 = tile * KT + 32 * KB * sub, r0 = 32 * KB * sub;
            if (!wave_on || k0 >= hi_max || k0 + 32 * KB <= lo_min) continue;
            at.pin();
            f32x16 s[RB][KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const v8 kx = att_row_frag<T, DP>(lk, at, r0 + 32 * kb, ks);
#pragma unroll
                    for (int i = 0; i < RB; ++i) {
                        if (ks == 0)
#pragma unroll
                            for (int e = 0; e < 16; ++e) s[i][kb][e] = 0.f;
                        s[i][kb] = mfma16(kx, qf[i][ks], s[i][kb]);
                    }
                }
            if (!asked) stage(tile + 1, buf ^ 1);
            asked = true;
            if (!(k0 >= lo_max && k0 + 32 * KB <= hi_min)) {
                // the rows' intervals are computed here, in the few tiles that straddle one, and hold no registers in the others
                AttArgsMem& m = *att_args();
                const int ln = att_lane();
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    const int n = att_div_g(m, row0 + 32 * i + (ln & 31));
                    int lo, hi;
                    att_range(m, n < qlen ? n : qlen - 1, qlen, klen, lo, hi);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int key = k0 + 32 * kb + acc_row(e, ln >> 5);
                            if (key < lo || key >= hi) s[i][kb][e] = -INFINITY;
                        }
                }
            }
            // The reference point of the exponentials moves only when a row's maximum has outgrown it by a factor of 2^8: until then the
            // sums stay within 2^8 of their scale, and the rescaling (every accumulator of the wave) is skipped.
            float mt[RB];
            bool grown = false;
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                mt[i] = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mt[i] = fmaxf(mt[i], s[i][kb][e]);
                grown = grown || mt[i] * c > mc[i] + 8.f;
            }
            if (__any(grown)) {
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    const float mn = fmaxf(mc[i], wave_half_xor_max(mt[i]) * c);   // a row's keys are in both lane halves: one point for both
                    const float alpha = __builtin_amdgcn_exp2f(mc[i] - mn);
                    mc[i] = mn;
                    l[i] *= alpha;
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][db][e] *= alpha;
                }
            }
            float p[RB][KB * 16];
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int e = 0; e < KB * 16; ++e) {
                    p[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e >> 4][e & 15], c, -mc[i]));
                    l[i] += p[i][e];                               // before its rounding: the backward pass divides by this sum
                }
#pragma unroll
            for (int ks = 0; ks < 2 * KB; ++ks) {
                v8 pf[RB];
#pragma unroll
                for (int i = 0; i < RB; ++i) pf[i] = att_pack<T>(p[i] + 8 * ks);
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const v8 vx = att_col_frag<T, DP>(lv, at, r0 + 16 * ks, db);
#pragma unroll
                    for (int i = 0; i < RB; ++i) acc[i][db] = mfma16(vx, pf[i], acc[i][db]);
                }
            }
        }
        if (!asked) stage(tile + 1, buf ^ 1);
    }

    AttArgsMem& m = *att_args();
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int row = row0 + 32 * i + r, n = att_div_g(m, row), head = hk * m.G + (row - n * m.G);
        if (n >= m.N) continue;
        const long long orow = ((long long)b * m.N + n) * m.H + head;
        const float sum = wave_half_xor_sum(l[i]);
        // by the interval, not by the sum: that is NaN where a visible score is, and such a row must not pass for one that sees nothing
        int lo, hi;
        att_range(m, n < qlen ? n : qlen - 1, qlen, klen, lo, hi);
        const bool some = n < qlen && lo < hi;
        if (m.splits > 1) {
            const long long rows = (long long)m.B * m.N * m.H;
            float* po = m.part + (split * rows + orow) * m.D;
#pragma unroll
            for (int db = 0; db < DB; ++db) att_store_block_f32(po, 32 * db, h, m.D, acc[i][db]);
            if (h == 0) {
                float* ml = m.part + (long long)m.splits * rows * m.D + (split * rows + orow) * 2;
                ml[0] = mc[i];
                ml[1] = some ? sum : -1.f;
            }
            continue;
        }
        T* o = (T*)m.out + orow * m.D;
        const float inv = some ? 1.f / sum : 0.f;
        if (some) {
#pragma unroll
            for (int db = 0; db < DB; ++db) att_store_block<T>(o, 32 * db, h, m.D, acc[i][db], inv);
        } else {                                                   // no visible key, or a row behind qlen
            for (int d = 8 * h; d < m.D; d += 16) *reinterpret_cast<u32x4*>(o + d) = u32x4{0, 0, 0, 0};
        }
        if (m.lse && h == 0) m.lse[((long long)b * m.H + head) * m.N + n] = some ? (mc[i] + log2f(sum)) * 0.69314718055994531f : -INFINITY;
    }
}

// joins the splits of a row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s. One workgroup per row: every lane of a wave holds the
// weight of one split (splits <= 64), thread (g, c) adds splits g, g + 8, .. of channels 4 c .. 4 c + 3, the eight sums meet in LDS.
// l_s is 0 where the row sees none of a split's keys, negative in every split where it sees no key at all, and NaN where a score is.
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
        if (!(ls <= 0.f)) ms = x.x;
    }
    const bool none = __shfl(ls, 0) < 0.f;
    float m = ms;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float f = ls <= 0.f ? -1.f : exp2f(ms - m);              // -1: the split has no part in the row
    float l = ls <= 0.f ? 0.f : f * ls;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
    if (threadIdx.x < 64) wt[lane] = f;
    __syncthreads();
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < a.D) {
#pragma unroll 4
        for (int k = g; k < a.splits; k += 8) {
            const float w = wt[k];
            if (!(w < 0.f)) {                                      // (a weight that vanished takes part: 0 times NaN is NaN)
                const f32x4 o = *reinterpret_cast<const f32x4*>(a.part + (k * rows + row) * a.D + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += w * o[j];
            }
        }
    }
    *reinterpret_cast<f32x4*>(&red[g][c]) = s;
    __syncthreads();
    const float inv = 1.f / l;                                     // of scores that are all -inf: 0 / 0
    if (threadIdx.x < a.D) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += red[k][threadIdx.x];
        ((T*)a.out)[row * a.D + threadIdx.x] = (T)(none ? 0.f : t * inv);
    }
    if (a.lse && threadIdx.x == 0) {
        const int h = (int)(row % a.H);
        const long long bn = row / a.H;
        const int n = (int)(bn % a.N);
        const long long b = bn / a.N;
        a.lse[(b * a.H + h) * a.N + n] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
}

struct AttPlan { int nw, rb, kt, tiles, splits; };

// One wave of 32 rows where that is all there are. Above, four waves: of one row block each, or of two at heads above 64,
// where a fragment read then serves two products and the registers allow it (4 x 4096 tokens, 16 heads of 128: 642 us with one, 560 us with
// two; heads of 64: 293 and 398 us), if the workgroups are enough for four rounds. Eight waves at heads of
// 33 to 64, halving the requests for keys, where that leaves the CUs as evenly filled (4 x 4096 tokens, 16 heads of 64: 334 us with four, 312
// with eight; 10240 tokens, 8 heads, 640 or 320 workgroups on 256 CUs: 285 and 320 us; with two waves 570 and 395). The keys are split
// where CUs would stand idle.
static AttPlan attention_plan(int B, int N, int M, int H, int Hk, int D) {
    const long long rows = (long long)N * (H / Hk), pairs = (long long)B * Hk, cus = svps_num_cus();
    AttPlan p;
    auto filled = [&](int nw) { return nw * ((pairs * ((rows + 32 * nw - 1) / (32 * nw)) + cus - 1) / cus); };     // waves on the fullest CU
    p.nw = rows <= 32 ? 1 : D > 32 && D <= 64 && filled(8) <= filled(4) ? 8 : 4;
    p.rb = D > 64 && pairs * ((rows + 255) / 256) >= 4 * cus ? 2 : 1;
    p.kt = p.nw == 1 ? 32 : 64;
    p.tiles = (int)((rows + 32 * p.nw * p.rb - 1) / (32 * p.nw * p.rb));
    const long long wgs = pairs * p.tiles, want = (p.nw == 1 ? 4LL : 2LL) * cus;
    const long long key_tiles = (M + p.kt - 1) / p.kt;
    long long s = wgs * 2 > want ? 1 : want / wgs;
    if (s > key_tiles / 4) s = key_tiles / 4;
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

template <typename T, int DP, int NW, int KT, int RB>
static int attention_launch(const AttArgs& a, hipStream_t stream) {
    static SvpsLdsAttr attr;
    constexpr int LDS = 4 * KT * DP * 2;
    const hipError_t e = attr.ensure((const void*)attention_fwd_kernel<T, DP, NW, KT, RB>, LDS);
    if (e != hipSuccess) return (int)e;
    const unsigned grid = (unsigned)((long long)a.B * a.Hk * a.tiles * a.splits);
    hipLaunchKernelGGL((attention_fwd_kernel<T, DP, NW, KT, RB>), dim3(grid), dim3(64 * NW), LDS, stream, a);
    return (int)hipGetLastError();
}

template <typename T, int DP>
static int attention_variant(const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    if (p.nw == 1) return attention_launch<T, DP, 1, 32, 1>(a, stream);
    if constexpr (DP == 128)
        if (p.rb == 2) return attention_launch<T, DP, 4, 64, 2>(a, stream);
    if constexpr (DP == 64)
        if (p.nw == 8) return attention_launch<T, DP, 8, 64, 1>(a, stream);
    return attention_launch<T, DP, 4, 64, 1>(a, stream);
}

template <typename T>
static int attention_dispatch(const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    const int rc = a.D <= 32 ? attention_variant<T, 32>(a, p, stream) : a.D <= 64 ? attention_variant<T, 64>(a, p, stream) : attention_variant<T, 128>(a, p, stream);
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
    const svps::AttPlan p = svps::attention_plan(B, N, M, H, Hk, D);
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
    const AttPlan p = attention_plan(B, N, M, H, Hk, D);
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
