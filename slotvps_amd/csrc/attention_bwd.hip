// Attention backward (attention.h has the layouts): the probabilities are computed again from q, k and the forward's log-sum-exp,
//   p = exp(s - lse),  delta_i = sum_d dO_id O_id,  dV = P^T dO,  dS = P * (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q.
//
// Two launches, no atomics, every sum in a fixed order:
//   att_stats_kernel    per packed row: lse in base 2, delta, visible interval - contiguous, so that the next one reads them as vectors
//   att_bwd_kernel      att_dkdv: a wave owns 32 keys (k, v as operand fragments in registers), walks over the rows that see them (q, dO
//                       in LDS);  att_dq: a wave owns 32 rows, walks over their keys like the forward
// That is 7 matrix products for the 5 of one joint kernel; the joint form would add dQ from many workgroups with atomics, whose order
// changes the result, or write every dS to memory (2 bytes per visible pair and head).
// Few tiles on either side: the walked range is split over workgroups that leave fp32 partial sums, added by att_add_kernel.
//
// P and dS are rounded to 16 bits once each, as operands of the products with dO, Q and K (the matrix instructions take 16 bits): beside the
// roundings of q, k, v and of the result they make a gradient 1.4 times as far off as its own rounding. Everything else is fp32. lse in fp32 is
// off by 2^-24 of itself, which every p of the row inherits: at scores of 10^4 2e-3, at 10^6 a fifth.
//
// Bound: the matrix products (10 D flop per visible pair, 14 D executed). Measured in bf16, all launches, flop counted as 10 D: 4 x 4096
// tokens, 16 heads of 128 1.75 ms = 785 TFLOP/s, causal over 4 key heads 0.96 ms = 717; 10240 tokens, 8 heads of 64 0.84 ms = 637, of 32
// 0.52 ms = 517 TFLOP/s; 5 x 100 tokens, 8 heads of 32 10.2 us. 4 x 4096 tokens, 16 heads of 40 1.15 ms, of 72 1.87 ms, of 96 1.95 ms.
#include "attention.h"
#include "../../include/slotvps_hip.h"

namespace svps {

// A wave takes 32 packed rows. delta = sum_d dO_id O_id is O's rounding to 16 bits away from sum_j p_ij dP_ij. Rows that spread over many keys do
// not notice (dS's own rounding is larger). Rows with nearly all their weight on one of many keys notice some: dQ is off by 1.4 times its own
// rounding at scores of standard deviation 1, by 2.2 at 4, by 3.5 at 16 (1000 tokens, 4 heads of 64); a delta from the products would cost two more
// products over all keys. Rows of few keys notice most: dS = P * (dP - delta) is then a small difference, of a single visible key
// zero (18 x 7 causal tokens, 2 / 1 heads of 96, against 64 bits: dQ 2.2 times as far off as its own rounding, as below 1.4 times). Where all keys
// that a wave's rows see lie within kStatKeys, delta is therefore the second sum (over the sum of p), from the same products that dQ and dK repeat.
constexpr int kStatKeys = 64;

template <typename T, int DP>
__global__ __launch_bounds__(256) void att_stats_kernel(AttArgs a) {
    typedef typename AttVec<T>::v8 v8;
    constexpr int L = DP / 8, PASS = 64 / L, KS = DP / 16;         // L lanes per row with 8 channels each, rows per pass
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = a.rows_pad / 128;
    const int pair = blockIdx.x / tiles, row0 = ((int)blockIdx.x - pair * tiles) * 128 + 32 * w;
    const int b = pair / a.Hk, hk = pair - b * a.Hk;
    const int qlen = att_qlen(a, b), klen = att_klen(a, b);
    const int n0 = att_div_g(a, row0);
    float delta = 0.f, lse2 = INFINITY;                            // of row row0 + r; exp2(. - inf) = 0: rows behind qlen and rows that see nothing
    int lo = 0, hi = 0;
    if (n0 < qlen) {
        const int row = row0 + r, n = att_div_g(a, row), head = hk * a.G + (row - n * a.G);
        const bool have = n < qlen;
        if (have) {
            att_range(a, n, qlen, klen, lo, hi);
            if (lo < hi) lse2 = a.lse[((long long)b * a.H + head) * a.N + n] * kLog2e;
        }
        int n1 = att_div_g(a, row0 + 31), lo_min, hi_max, tmp;
        n1 = n1 < qlen ? n1 : qlen - 1;
        att_range(a, n0, qlen, klen, lo_min, tmp);
        att_range(a, n1, qlen, klen, tmp, hi_max);
        if (hi_max - lo_min <= kStatKeys) {
            const T* qp = (const T*)a.q + b * a.sqb + n * a.sqn + head * a.sqh;
            const T* dp = (const T*)a.dout + b * a.sdb + n * a.sdn + head * a.sdh;
            const T* kp = (const T*)a.k + b * a.skb + hk * a.skh;
            const T* vp = (const T*)a.v + b * a.svb + hk * a.svh;
            const float c = a.scale * kLog2e;
            float sum = 0.f;
            auto piece = [&](const T* x, bool on, int d) __attribute__((always_inline)) {
                u32x4 y = {0, 0, 0, 0};
                if (on && d < a.D) y = *reinterpret_cast<const u32x4*>(x + d);
                return __builtin_bit_cast(v8, y);
            };
            for (int k0 = lo_min; k0 < hi_max; k0 += 32) {
                const int kr = k0 + r < hi_max ? k0 + r : hi_max - 1;
                f32x16 s, g;
#pragma unroll
                for (int i = 0; i < 16; ++i) { s[i] = 0.f; g[i] = 0.f; }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int d = 16 * ks + 8 * h;
                    s = mfma16(piece(kp + kr * a.skn, true, d), piece(qp, have, d), s);
                    g = mfma16(piece(vp + kr * a.svn, true, d), piece(dp, have, d), g);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = k0 + acc_row(i, h);
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2));
                    if (key >= lo && key < hi) {
                        sum += p;
                        delta = fmaf(p, g[i], delta);
                    }
                }
            }
            delta += __shfl_xor(delta, 32);
            sum += __shfl_xor(sum, 32);
            delta = sum == 0.f ? 0.f : delta / sum;                // the sum is 1 but for the roundings of lse: of one key, delta is dP to the bit
        } else {
#pragma unroll 4
            for (int q = 0; q < 32; q += PASS) {
                const int rr = row0 + q + lane / L, m = att_div_g(a, rr), hd = hk * a.G + (rr - m * a.G), d = 8 * (lane % L);
                float t = 0.f;
                if (m < qlen && d < a.D) {
                    const v8 x = *reinterpret_cast<const v8*>((const T*)a.dout + b * a.sdb + m * a.sdn + hd * a.sdh + d);
                    const v8 y = *reinterpret_cast<const v8*>((const T*)a.out_in + (((long long)b * a.N + m) * a.H + hd) * a.D + d);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t += (float)x[j] * (float)y[j];
                }
#pragma unroll
                for (int o = 1; o < L; o <<= 1) t += __shfl_xor(t, o);
                t = __shfl(t, ((r - q) & (PASS - 1)) * L);          // row q + i stands in lanes L i ..
                if (r >= q && r < q + PASS) delta = t;
            }
        }
    }
    if (h == 0) {
        const long long prow = (long long)pair * a.rows_pad + row0 + r;
        a.stat_lse2[prow] = lse2;
        a.stat_delta[prow] = delta;
        a.stat_lo[prow] = lo;
        a.stat_hi[prow] = hi;
    }
}

// dQ of 128 packed rows: a wave owns 32 rows and walks over their keys
template <typename T, int DP>
__device__ __forceinline__ void att_dq(const AttArgs& a, const int id, char* smem) {
    typedef typename AttVec<T>::v8 v8;
    constexpr int KT = 64, KS = DP / 16, DB = DP / 32, KB = KT / 32, TILE = KT * DP * 2, NW = 4;
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = a.B * a.Hk;
    const int rest = id / pairs, pair = att_pair(id, rest, pairs);
    const int t = a.tiles - 1 - rest % a.tiles, split = rest / a.tiles;
    const int b = pair / a.Hk, hk = pair - b * a.Hk;
    const int qlen = att_qlen(a, b), klen = att_klen(a, b);
    const int row0 = (t * NW + w) * 32, row = row0 + r;
    const int n = att_div_g(a, row);
    const int head = hk * a.G + (row - n * a.G);
    const bool have = n < qlen;
    const int wg0 = att_div_g(a, t * NW * 32);
    int wg1 = att_div_g(a, t * NW * 32 + NW * 32 - 1);
    wg1 = wg1 < qlen ? wg1 : qlen - 1;
    int tb = 0, te = 0, lo_min = 0, hi_min = 0, lo_max = 0, hi_max = 0, tmp;
    const int wn0 = att_div_g(a, row0);
    const bool wave_on = wn0 < qlen;
    if (wg0 < qlen) {
        int lo_wg, hi_wg;
        att_range(a, wg0, qlen, klen, lo_wg, tmp);
        att_range(a, wg1, qlen, klen, tmp, hi_wg);
        int wn1 = att_div_g(a, row0 + 31);
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
    const long long prow = (long long)pair * a.rows_pad + row;     // rows_pad is a multiple of 128
    const float lse2 = a.stat_lse2[prow], delta = a.stat_delta[prow];
    const int lo = a.stat_lo[prow], hi = a.stat_hi[prow];

    v8 qf[KS], df[KS];
    {
        const T* qp = (const T*)a.q + b * a.sqb + n * a.sqn + head * a.sqh;
        const T* dp = (const T*)a.dout + b * a.sdb + n * a.sdn + head * a.sdh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 16 * ks + 8 * h;
            u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            if (have && d < a.D) {
                x = *reinterpret_cast<const u32x4*>(qp + d);
                y = *reinterpret_cast<const u32x4*>(dp + d);
            }
            qf[ks] = __builtin_bit_cast(v8, x);
            df[ks] = __builtin_bit_cast(v8, y);
        }
    }
    AttTile<DP, KT, NW, kAttK> tk;
    AttTile<DP, KT, NW, kAttV> tv;
    tk.init((const T*)a.k + b * a.skb + hk * a.skh, a, w, lane);
    tv.init((const T*)a.v + b * a.svb + hk * a.svh, a, w, lane);
    auto stage = [&](int tile, int buf) __attribute__((always_inline)) {
        char* lk = smem + buf * 2 * TILE;
        tk.stage(tile, klen, lk, w);
        tv.stage(tile, klen, lk + TILE, w);
    };
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
    const float c = a.scale * kLog2e;
    AttLane<DP> at(lane);
    if (tb < te) stage(tb, 0);
    for (int tile = tb; tile < te; ++tile) {
        const int buf = (tile - tb) & 1;
        wait_vm<0>();
        wg_barrier();
        const int k0 = tile * KT;
        if (!wave_on || k0 >= hi_max || k0 + KT <= lo_min) {
            if (tile + 1 < te) stage(tile + 1, buf ^ 1);
            continue;
        }
        const char* lk = smem + buf * 2 * TILE;
        const char* lv = lk + TILE;
        at.pin();
        const bool whole = k0 >= lo_max && k0 + KT <= hi_min;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = mfma16(att_row_frag<T, DP>(lk, at, 32 * kb, ks), qf[ks], s);
                dp = mfma16(att_row_frag<T, DP>(lv, at, 32 * kb, ks), df[ks], dp);
            }
            if (kb == 0 && tile + 1 < te) stage(tile + 1, buf ^ 1);
            float ds[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2));
                ds[i] = p * (dp[i] - delta);
            }
            if (!whole) {
                asm volatile("");                                  // a branch, not 16 selects in every tile
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = k0 + 32 * kb + acc_row(i, h);
                    if (key < lo || key >= hi) ds[i] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const v8 pf = att_pack<T>(ds + 8 * u);
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[db] = mfma16(att_col_frag<T, DP>(lk, at, 32 * kb + 16 * u, db), pf, acc[db]);
            }
        }
    }
    AttArgsMem& m = *att_args();
    if (n >= m.N) return;
    if (lo >= hi) {                                                // behind qlen, or sees nothing: its weights are 0, but 0 times a key that is NaN is not
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
    }
    const long long orow = ((long long)b * m.N + n) * m.H + hk * m.G + (row - n * m.G);
    if (m.splits > 1) {
        float* po = m.part + (split * ((long long)m.B * m.N * m.H) + orow) * m.D;
#pragma unroll
        for (int db = 0; db < DB; ++db) att_store_block_f32(po, 32 * db, h, m.D, acc[db]);
        return;
    }
    T* o = (T*)m.dq + orow * m.D;
#pragma unroll
    for (int db = 0; db < DB; ++db) att_store_block<T>(o, 32 * db, h, m.D, acc[db], m.scale);
}

// tokens [n0, n1) that see a key of [k0, k1): their frame is not before the first key's, and not `window` or more behind the last key's
template <typename A>
__device__ __forceinline__ void att_seen_by(const A& a, int k0, int k1, int qlen, int klen, int& n0, int& n1) {
    n0 = 0;
    n1 = k0 < klen ? qlen : 0;
    if (a.frame > 0 && n1 > 0) {
        k1 = k1 < klen ? k1 : klen;
        const long long off = (long long)klen - qlen;
        const long long first = (long long)(k0 / a.frame) * a.frame - off;
        if (first > 0) n0 = first < qlen ? (int)first : qlen;
        if (a.window > 0) {
            const long long last = ((long long)((k1 - 1) / a.frame) + a.window) * a.frame - off;
            if (last < n1) n1 = last > 0 ? (int)last : 0;
        }
    }
}

// dK, dV of 128 keys: a wave owns 32 keys, their k and v stay in registers as operand fragments (at DP = 128 the sums and they are 192 of 256
// registers: one block of scores at a time, fragments one step ahead, two of v's eight fragments in LDS - with all in registers a few
// values went to scratch, whose loads stand in one queue with the tiles on their way). (lse, delta) of a tile's rows come by LDS-DMA with the rows.
template <typename T, int DP>
__device__ __forceinline__ void att_dkdv(const AttArgs& a, const int id, char* smem) {
    typedef typename AttVec<T>::v8 v8;
    constexpr int KS = DP / 16, DB = DP / 32, QT = 64, TILE = QT * DP * 2, NW = 4, BUF = 2 * TILE + 512, VR = DP == 128 ? 6 : KS;
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = a.B * a.Hk;
    const int rest = id / pairs, pair = att_pair(id, rest, pairs);
    const int t = rest / a.k_splits, split = rest - t * a.k_splits;    // early keys are seen by the most rows: longest first
    const int b = pair / a.Hk, hk = pair - b * a.Hk;
    const int qlen = att_qlen(a, b), klen = att_klen(a, b);
    const int wk0 = t * 128, k0 = wk0 + 32 * w, key = k0 + r;

    int n0, n1;
    att_seen_by(a, wk0, wk0 + 128, qlen, klen, n0, n1);
    int tb = 0, te = 0;
    if (n0 < n1) {
        tb = (int)((long long)n0 * a.G / QT);
        te = (int)(((long long)n1 * a.G + QT - 1) / QT);
    }
    if (a.k_splits > 1) {
        const int per = (te - tb + a.k_splits - 1) / a.k_splits;
        tb += split * per;
        te = tb + per < te ? tb + per : te;
    }

    v8 kf[KS], vf[VR];
    char* vkeep = smem + 2 * BUF + w * (KS - VR) * 1024 + lane * 16;
    {
        const T* kp = (const T*)a.k + b * a.skb + hk * a.skh + (long long)key * a.skn;
        const T* vp = (const T*)a.v + b * a.svb + hk * a.svh + (long long)key * a.svn;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 16 * ks + 8 * h;
            u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            if (key < klen && d < a.D) {
                x = *reinterpret_cast<const u32x4*>(kp + d);
                y = *reinterpret_cast<const u32x4*>(vp + d);
            }
            kf[ks] = __builtin_bit_cast(v8, x);
            if (ks < VR) vf[ks < VR ? ks : 0] = __builtin_bit_cast(v8, y);
            else *reinterpret_cast<u32x4*>(vkeep + (ks - VR) * 1024) = y;     // read by the lane that wrote it
        }
    }
    const long long pbase = (long long)pair * a.rows_pad;
    AttTile<DP, QT, NW, kAttQ> tq;
    AttTile<DP, QT, NW, kAttDout> td;
    tq.init((const T*)a.q + b * a.sqb + hk * a.G * a.sqh, a, w, lane);
    td.init((const T*)a.dout + b * a.sdb + hk * a.G * a.sdh, a, w, lane);
    auto stage = [&](int tile, int buf) __attribute__((always_inline)) {
        char* lq = smem + buf * BUF;
        tq.stage(tile, qlen * a.G, lq, w);
        td.stage(tile, qlen * a.G, lq + TILE, w);
        if (w < 2) {                                               // 64 rows of lse2 (wave 0) and delta (wave 1); rows_pad is a multiple of 128
            const float* src = (w ? a.stat_delta : a.stat_lse2) + pbase + tile * QT;
            dma_off4(dma_base((const char*)src), att_lane() * 4, lq + 2 * TILE + 256 * w);
        }
    };
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[db][i] = 0.f; dv[db][i] = 0.f; }
    const float c = a.scale * kLog2e;
    AttLane<DP> at(lane);
    if (tb < te) stage(tb, 0);
    for (int tile = tb; tile < te; ++tile) {
        const int buf = (tile - tb) & 1;
        wait_vm<0>();
        wg_barrier();
        if (tile + 1 < te) stage(tile + 1, buf ^ 1);
        const char* lq = smem + buf * BUF;
        const char* ld = lq + TILE;
#pragma unroll 1
        for (int qb = 0; qb < QT / 32; ++qb) {
            const int row0 = tile * QT + 32 * qb;
            // interval bounds never fall along the rows: those of the block's first and last token decide whether comparisons are needed, or anything
            const int nf = att_div_g(a, row0), nl = att_div_g(a, row0 + 31);
            if (k0 >= klen || nf >= qlen) continue;
            bool whole = nl < qlen && k0 + 32 <= klen;
            if (a.frame > 0) {
                int lo_f, hi_f, lo_l, hi_l;
                att_range(a, nf, qlen, klen, lo_f, hi_f);
                att_range(a, nl < qlen ? nl : qlen - 1, qlen, klen, lo_l, hi_l);
                if (k0 + 32 <= lo_f || k0 >= hi_l) continue;
                whole = whole && k0 >= lo_l && k0 + 32 <= hi_f;
            }
            at.pin();
            const float* st = reinterpret_cast<const float*>(lq + 2 * TILE) + 32 * qb + 4 * h;
            v8 pf[2], sf[2];
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = 0.f; }
            v8 qa = att_row_frag<T, DP>(lq, at, 32 * qb, 0), da = att_row_frag<T, DP>(ld, at, 32 * qb, 0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {                      // operands one step ahead and no further: at DP = 128 there are no registers for more
                v8 qn, dn;
                if (ks + 1 < KS) {
                    qn = att_row_frag<T, DP>(lq, at, 32 * qb, ks + 1);
                    dn = att_row_frag<T, DP>(ld, at, 32 * qb, ks + 1);
                }
                const v8 vv = ks < VR ? vf[ks < VR ? ks : 0] : *reinterpret_cast<const v8*>(vkeep + (ks - VR) * 1024);
                if (DP == 128) __builtin_amdgcn_sched_barrier(0);
                s = mfma16(qa, kf[ks], s);
                dp = mfma16(da, vv, dp);
                if (DP == 128) __builtin_amdgcn_sched_barrier(0);
                qa = qn;
                da = dn;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(st + 8 * e);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * e + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * e + j], c, -ls[j]));
            }
            if (!whole) {
                AttArgsMem& m = *att_args();                       // (also keeps this a branch instead of 16 selects in every block)
                typedef int i32x4 __attribute__((ext_vector_type(4)));
                const int h4 = (att_lane() >> 5) * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const i32x4 lo = *reinterpret_cast<const i32x4*>(m.stat_lo + pbase + row0 + (8 * e + h4));
                    const i32x4 hi = *reinterpret_cast<const i32x4*>(m.stat_hi + pbase + row0 + (8 * e + h4));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (key < lo[j] || key >= hi[j]) s[4 * e + j] = 0.f;
                }
            }
            float p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = s[i];
#pragma unroll
            for (int u = 0; u < 2; ++u) pf[u] = att_pack<T>(p + 8 * u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x4 de = *reinterpret_cast<const f32x4*>(st + 64 + 8 * e);
#pragma unroll
                for (int j = 0; j < 4; ++j) p[4 * e + j] *= dp[4 * e + j] - de[j];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) sf[u] = att_pack<T>(p + 8 * u);
            if (DP == 128) __builtin_amdgcn_sched_barrier(0);     // one block of scores at a time in registers
            v8 dc = att_col_frag<T, DP>(ld, at, 32 * qb, 0), qc = att_col_frag<T, DP>(lq, at, 32 * qb, 0);
#pragma unroll
            for (int i = 0; i < 2 * DB; ++i) {
                const int u = i / DB, db = i % DB, un = (i + 1) / DB, dn = (i + 1) % DB;
                v8 dx, qx;
                if (i + 1 < 2 * DB) {
                    dx = att_col_frag<T, DP>(ld, at, 32 * qb + 16 * un, dn);
                    qx = att_col_frag<T, DP>(lq, at, 32 * qb + 16 * un, dn);
                }
                if (DP == 128) __builtin_amdgcn_sched_barrier(0);
                dv[db] = mfma16(dc, pf[u], dv[db]);
                dk[db] = mfma16(qc, sf[u], dk[db]);
                if (DP == 128) __builtin_amdgcn_sched_barrier(0);
                dc = dx;
                qc = qx;
            }
        }
    }
    AttArgsMem& m = *att_args();
    if (key >= m.M) return;
    att_seen_by(m, key, key + 1, qlen, klen, n0, n1);
    if (n0 >= n1) {                                                // behind klen, or seen by no row: 0 times a row that is NaN is not 0
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) { dk[db][i] = 0.f; dv[db][i] = 0.f; }
    }
    const long long orow = ((long long)b * m.M + key) * m.Hk + hk;
    if (m.k_splits > 1) {
        const long long rows = (long long)m.B * m.M * m.Hk;
        float* pk = m.k_part + (split * rows + orow) * m.D;
        float* pv = pk + (long long)m.k_splits * rows * m.D;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            att_store_block_f32(pk, 32 * db, h, m.D, dk[db]);
            att_store_block_f32(pv, 32 * db, h, m.D, dv[db]);
        }
        return;
    }
    T* ok = (T*)m.dk + orow * m.D;
    T* ov = (T*)m.dv + orow * m.D;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        att_store_block<T>(ok, 32 * db, h, m.D, dk[db], m.scale);
        att_store_block<T>(ov, 32 * db, h, m.D, dv[db], 1.f);
    }
}

// one launch for both: they are independent, the workgroups of dQ fill what those of dK, dV leave idle
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void att_bwd_kernel(AttArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int n = a.B * a.Hk * a.k_tiles * a.k_splits;
    if ((int)blockIdx.x < n) att_dkdv<T, DP>(a, blockIdx.x, smem);
    else att_dq<T, DP>(a, blockIdx.x - n, smem);
}

// out = f * sum over splits, four values per thread, splits in order (count % 4 == 0: D % 8 == 0)
template <typename T>
__global__ __launch_bounds__(256) void att_add_kernel(const float* part, T* out, long long count, int splits, float f) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= count) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < splits; ++k) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(part + k * count + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += x[j];
    }
    typename AttVec<T>::v4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (T)(s[j] * f);
    *reinterpret_cast<typename AttVec<T>::v4*>(out + i) = o;
}

int attention_check(const void* const* ptrs, int np, const long long* const* strides, int ns, int B, int N, int M, int H, int Hk, int D,
                    int frame, int window, float scale, int dtype);

struct AttBwdPlan {
    int q_tiles, q_splits, k_tiles, k_splits, rows_pad;
    size_t stat_bytes, q_part_bytes, k_part_bytes;
};

static AttBwdPlan attention_bwd_plan(int B, int N, int M, int H, int Hk, int D) {
    AttBwdPlan p;
    const long long rows = (long long)N * (H / Hk), pairs = (long long)B * Hk, want = 2LL * svps_num_cus();
    p.q_tiles = (int)((rows + 127) / 128);
    p.k_tiles = (M + 127) / 128;
    p.rows_pad = p.q_tiles * 128;
    auto pick = [&](long long wgs, long long steps) {
        long long s = wgs * 2 > want ? 1 : want / wgs;
        if (s > steps / 4) s = steps / 4;
        if (s > 32) s = 32;
        return s < 1 ? 1 : (int)s;
    };
    p.q_splits = pick(pairs * p.q_tiles, (M + 63) / 64);
    // dK / dV: the split that is done first by a model of workgroups that all see every row, in microseconds: rounds of 64-row steps
    // (1.3 at DP = 128 with one workgroup per CU, about the same for two of the smaller sizes) plus the partial sums' way to memory
    // and back at 4 TB/s. (In causal order the tiles differ; the longest go first, and a split halves the longest.)
    {
        const long long wgs = pairs * p.k_tiles, slots = 2LL * svps_num_cus(), steps = (rows + 63) / 64;
        double best = 0.0;
        p.k_splits = 1;
        for (int s = 1; s <= 32 && (s == 1 || steps / s >= 4); ++s) {
            const double t = (double)((wgs * s + slots - 1) / slots) * (double)((steps + s - 1) / s) * 1.3 +
                             (s > 1 ? 5.0 + (double)s * B * M * Hk * D * 16.0 / 4e6 : 0.0);
            if (s == 1 || t < best) { best = t; p.k_splits = s; }
        }
    }
    p.stat_bytes = (size_t)pairs * p.rows_pad * 4 * sizeof(float);
    p.q_part_bytes = p.q_splits > 1 ? (size_t)p.q_splits * B * N * H * D * sizeof(float) : 0;
    p.k_part_bytes = p.k_splits > 1 ? (size_t)p.k_splits * B * M * Hk * D * 2 * sizeof(float) : 0;
    return p;
}

template <typename T, int DP>
static int attention_bwd_launch(const AttArgs& a, const AttBwdPlan& p, hipStream_t stream) {
    static SvpsLdsAttr attr;
    constexpr int LDS = 2 * (2 * 64 * DP * 2 + 512) + (DP == 128 ? 8192 : 0);     // two pairs of 64-row tiles; for dK and dV their (lse, delta) and kept fragments
    hipError_t e = attr.ensure((const void*)att_bwd_kernel<T, DP>, LDS);
    if (e != hipSuccess) return (int)e;
    const long long pairs = (long long)a.B * a.Hk;
    hipLaunchKernelGGL((att_stats_kernel<T, DP>), dim3((unsigned)(pairs * (a.rows_pad / 128))), dim3(256), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    const unsigned grid = (unsigned)(pairs * ((long long)a.k_tiles * a.k_splits + (long long)a.tiles * a.splits));
    hipLaunchKernelGGL((att_bwd_kernel<T, DP>), dim3(grid), dim3(256), LDS, stream, a);
    e = hipGetLastError();
    auto add = [&](const float* part, void* out, long long count, int splits, float f) {
        if (e != hipSuccess) return;
        hipLaunchKernelGGL(att_add_kernel<T>, dim3((unsigned)((count / 4 + 255) / 256)), dim3(256), 0, stream, part, (T*)out, count, splits, f);
        e = hipGetLastError();
    };
    if (a.k_splits > 1) {
        const long long count = (long long)a.B * a.M * a.Hk * a.D;
        add(a.k_part, a.dk, count, a.k_splits, a.scale);
        add(a.k_part + a.k_splits * count, a.dv, count, a.k_splits, 1.f);
    }
    if (a.splits > 1) add(a.part, a.dq, (long long)a.B * a.N * a.H * a.D, a.splits, a.scale);
    return (int)e;
}

}  // namespace svps

extern "C" size_t svps_attention_bwd_workspace_bytes(int B, int N, int M, int H, int Hk, int D) {
    if (B <= 0 || N <= 0 || M <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0) return 0;
    const svps::AttBwdPlan p = svps::attention_bwd_plan(B, N, M, H, Hk, D);
    return p.stat_bytes + p.q_part_bytes + p.k_part_bytes;
}

extern "C" int svps_attention_bwd(const void* dout, const long long* sd, const void* q, const long long* sq, const void* k, const long long* sk,
                                  const void* v, const long long* sv, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                  const int* qlens, const int* klens, void* workspace, size_t workspace_bytes, int B, int N, int M, int H,
                                  int Hk, int D, int frame, int window, float scale, int dtype, void* stream) {
    using namespace svps;
    const void* ptrs[] = {dout, q, k, v, out, dq, dk, dv, workspace};
    const long long* st[] = {sd, sq, sk, sv};
    if (!lse) return SVPS_ERR_BAD_ARG;
    const int rc = attention_check(ptrs, 9, st, 4, B, N, M, H, Hk, D, frame, window, scale, dtype);
    if (rc) return rc;
    const AttBwdPlan p = attention_bwd_plan(B, N, M, H, Hk, D);
    if (workspace_bytes < p.stat_bytes + p.q_part_bytes + p.k_part_bytes) return SVPS_ERR_WORKSPACE;
    AttArgs a = {};
    a.q = q; a.k = k; a.v = v; a.dout = dout; a.out_in = out; a.lse = const_cast<float*>(lse);
    a.dq = dq; a.dk = dk; a.dv = dv; a.qlens = qlens; a.klens = klens;
    a.sqb = sq[0]; a.sqn = sq[1]; a.sqh = sq[2]; a.skb = sk[0]; a.skn = sk[1]; a.skh = sk[2];
    a.svb = sv[0]; a.svn = sv[1]; a.svh = sv[2]; a.sdb = sd[0]; a.sdn = sd[1]; a.sdh = sd[2];
    const size_t rows = (size_t)B * Hk * p.rows_pad;
    a.stat_lse2 = (float*)workspace;
    a.stat_delta = a.stat_lse2 + rows;
    a.stat_lo = (int*)(a.stat_delta + rows);
    a.stat_hi = a.stat_lo + rows;
    a.part = (float*)((char*)workspace + p.stat_bytes);
    a.k_part = (float*)((char*)workspace + p.stat_bytes + p.q_part_bytes);
    a.rows_pad = p.rows_pad;
    a.tiles = p.q_tiles; a.splits = p.q_splits; a.k_tiles = p.k_tiles; a.k_splits = p.k_splits;
    a.B = B; a.N = N; a.M = M; a.H = H; a.Hk = Hk; a.G = H / Hk; a.D = D; a.frame = frame; a.window = window;
    a.scale = scale;
    a.gmagic = a.G > 1 ? (unsigned)(0x100000000ULL / a.G) + 1 : 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == SVPS_DTYPE_BF16)
        return D <= 32 ? attention_bwd_launch<__bf16, 32>(a, p, s) : D <= 64 ? attention_bwd_launch<__bf16, 64>(a, p, s) : attention_bwd_launch<__bf16, 128>(a, p, s);
    return D <= 32 ? attention_bwd_launch<_Float16, 32>(a, p, s) : D <= 64 ? attention_bwd_launch<_Float16, 64>(a, p, s) : attention_bwd_launch<_Float16, 128>(a, p, s);
}
