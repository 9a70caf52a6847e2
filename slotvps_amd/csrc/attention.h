// Shared by attention_fwd.hip and attention_bwd.hip: attention of 16-bit queries over 16-bit keys and values with shared key heads.
//
//   s_ij = scale q_i . k_j for lo_i <= j < hi_i,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//
// The G = H / Hk query heads of one key head are packed into the row axis: row rr of a (batch entry, key head) pair is token rr / G, head
// G * hk + rr % G. A tile of rows then reads its keys and values once for all G heads, a single query of G heads is G rows of one tile, and
// the gradients of a shared head sum inside the matrix products.
//
// Visible keys are an interval per row, from lengths and frame order alone (no mask is read): [0, klen) without order; with `frame` > 0
// tokens of one frame see each other and all earlier frames, `window` > 0 only the last `window` frames, their own counted. The last
// query stands at the last key. lo and hi never fall along the rows, so tiles outside [lo of the first row, hi of the last) are never
// visited and only tiles that straddle a bound pay for comparisons.
//
// Matrix operands (v_mfma_f32_32x32x16): the scores are computed TRANSPOSED, S^T = K Q^T, so a lane owns one query row and the softmax
// runs inside the lane (one exchange with lane ^ 32). The accumulator then holds, for a step of 16 keys, keys 4h + {0..3} and 8 + 4h + {0..3}
// in lane half h; the contraction index of the next product is laid out in that same order (its other operand comes from LDS through the
// hardware transpose, which takes any row order), so probabilities go from accumulator to operand without crossing lanes.
//
// LDS tiles: rows of DP 16-bit channels (DP = head size padded to 32, 64 or 128 with zeros), 16-byte chunk c of row r at position
// c ^ att_swz(r): fragment reads along a chunk column (16 rows) and transposed reads (4 rows x 4 chunks) both touch 16 different slots.
#pragma once
#include "common.h"

namespace svps {

struct AttArgs {
    const void* q; const void* k; const void* v; const void* dout;
    void* out;                                  // forward: [B, N, H, D]
    void* dq; void* dk; void* dv;               // contiguous [B, N, H, D], [B, M, Hk, D]
    const void* out_in;                         // backward: the forward's output
    float* lse;                                 // [B, H, N]
    long long sqb, sqn, sqh, skb, skn, skh, svb, svn, svh, sdb, sdn, sdh;
    const int* qlens; const int* klens;
    float* part; float* k_part;                 // partial sums of splits (backward: dQ | dK, dV)
    float* stat_lse2; float* stat_delta; int* stat_lo; int* stat_hi;   // backward: per packed row, [B * Hk][rows_pad]
    int B, N, M, H, Hk, G, D, frame, window, splits, tiles, k_splits, k_tiles, rows_pad;
    unsigned gmagic;                            // floor(2^32 / G) + 1
    float scale;
};

// the lane's number, computed where it stands (a value kept from the start would hold a register through the main loop)
__device__ __forceinline__ int att_lane() {
    int x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
}

// The kernel's arguments (its only parameter) read again from memory: for code behind or beside the main loop, whose values would otherwise
// stand in scalar registers all through it (and push each other out of them).
typedef const AttArgs __attribute__((address_space(4))) AttArgsMem;
__device__ __forceinline__ AttArgsMem* att_args() {
    AttArgsMem* p = (AttArgsMem*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

__device__ __forceinline__ int att_qlen(const AttArgs& a, int b) {
    if (!a.qlens) return a.N;
    const int n = a.qlens[b];
    return n < 0 ? 0 : (n > a.N ? a.N : n);
}
__device__ __forceinline__ int att_klen(const AttArgs& a, int b) {
    if (!a.klens) return a.M;
    const int n = a.klens[b];
    return n < 0 ? 0 : (n > a.M ? a.M : n);
}

// row / G without a division: the product with floor(2^32 / G) + 1 is never short and at most one too far
template <typename A>
__device__ __forceinline__ int att_div_g(const A& a, int row) {
    if (a.G == 1) return row;
    int n = (int)__umulhi((unsigned)row, a.gmagic);
    return n - ((long long)n * a.G > row ? 1 : 0);
}

// Workgroups go round the 8 XCDs in order of their number. Each row of `pairs` numbers is turned by one against the last, so that an XCD
// meets every pair: fixed to one pair, the XCDs of a short batch entry stand idle (two entries of 4097 and 2000 tokens: 158 us, turned
// 113 us). The tiles of a pair that an XCD holds at a time walk over the same keys together and share them in its L2 as before.
__device__ __forceinline__ int att_pair(int id, int rest, int pairs) { return (int)(((long long)id + rest) % pairs); }

__device__ __forceinline__ int floor_div(int x, int d) {
    const int q = x / d;
    return q - ((x - q * d) < 0 ? 1 : 0);
}

// visible keys [lo, hi) of token n (0 <= n < qlen)
template <typename A>
__device__ __forceinline__ void att_range(const A& a, int n, int qlen, int klen, int& lo, int& hi) {
    lo = 0;
    hi = klen;
    if (a.frame > 0) {
        const int p = n + klen - qlen;
        const int f = a.frame == 1 ? p : floor_div(p, a.frame);
        const long long end = ((long long)f + 1) * a.frame;
        hi = end < klen ? (int)end : klen;
        if (a.window > 0 && f >= a.window) lo = (f - a.window + 1) * a.frame;
        if (hi < 0) hi = 0;
        if (lo > hi) lo = hi;
    }
}

template <int DP> __device__ __forceinline__ int att_swz(int row) {
    if constexpr (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (DP == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
}

static __device__ __attribute__((aligned(16))) uint32_t g_att_zero[4];       // never written: the source of padded rows and channels

// LDS-DMA: 64 lanes x 16 (4) bytes to lds_base + lane * 16 (4), with a wave-uniform base (64-bit, scalar registers) and a 32-bit lane offset
// below 2 GiB, or with a 64-bit address per lane. Written as instructions: behind the builtin the compiler knows of a pending write to LDS
// and waits for ALL of them in front of every transposed read, i.e. for the tile it has just asked for. Nothing is returned to a register;
// the waits are the ones in the code (wait_vm in front of the barrier that hands a tile over). They are ordered against the barriers
// (volatile) and free against LDS reads, which only touch the other buffer between two barriers. The address unit takes 16 cycles for
// each: issued in a row behind a barrier they can hold every wave of the CU up. The forward kernel and dQ ask for the next tile behind
// their first products (4097 causal tokens, 16 / 4 heads of 128: 110 -> 100 us forward); dK / dV and the products of linear_act ask right
// behind the barrier (behind the products: 4097 tokens 300 -> 322 us, 8192^3 935 -> 970 us).
__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(p));        // the low half of a flat address into LDS
}
__device__ __forceinline__ u32x4 dma_base(const char* base) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu), 0x7fffffffu, 0x00020000u};
}
__device__ __forceinline__ void dma_off(u32x4 base, uint32_t lane_off, const char* lds_base) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds_address(lds_base)), "v"(lane_off), "s"(base));
}
__device__ __forceinline__ void dma_off4(u32x4 base, uint32_t lane_off, const char* lds_base) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds_address(lds_base)), "v"(lane_off), "s"(base));
}
__device__ __forceinline__ void dma_ptr(const char* src, const char* lds_base) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds_address(lds_base)), "v"(src));
}

template <typename T> struct AttVec;
template <> struct AttVec<__bf16> { typedef bf16x8 v8; typedef bf16x4 v4; };
template <> struct AttVec<_Float16> { typedef f16x8 v8; typedef f16x4 v4; };

// ROWS packed rows of a [tokens, heads, D] operand into an LDS tile by 16-byte LDS-DMA. Packed row rr is token rr / G, head rr % G of the
// group (keys and values: G = 1). For whole tiles of DP channels a lane's offsets are the same in every tile and only the wave-uniform
// base moves (no address arithmetic in the loop); rows behind the last valid one and padded channels take zeros on a slower path - what
// stands behind a length must not reach a product, 0 * NaN included.
enum { kAttQ, kAttK, kAttV, kAttDout };
template <int DP, int ROWS, int NW, int OP, bool HOLD = true>
struct AttTile {
    static constexpr int CH = DP / 8, RPP = 64 / CH, PIECES = ROWS / RPP, N = PIECES / NW, LEAP = RPP * NW;
    static constexpr int NOFF = LEAP % 16 == 0 ? 1 : N;     // pieces 16 k rows apart have the same swizzle: one offset, the rest is uniform
    static_assert(PIECES % NW == 0, "every wave stages the same number of pieces");
    const char* base;
    long long step, leap;                       // bytes from tile to tile, from piece to piece
    uint32_t off[NOFF];                         // HOLD = false: computed per tile, for the kernel whose registers are full
    static_assert(HOLD || NOFF == 1, "");
    bool quick;
    template <typename A> static __device__ __forceinline__ long long token(const A& a) { return 2 * (OP == kAttQ ? a.sqn : OP == kAttK ? a.skn : OP == kAttV ? a.svn : a.sdn); }
    template <typename A> static __device__ __forceinline__ long long head(const A& a) { return OP == kAttQ ? 2 * a.sqh : OP == kAttDout ? 2 * a.sdh : 0; }
    template <typename A> static __device__ __forceinline__ int group(const A& a) { return OP == kAttQ || OP == kAttDout ? a.G : 1; }
    template <typename A> static __device__ __forceinline__ uint32_t offset(const A& a, int i, int w, int lane) {
        const int row = (i * NW + w) * RPP + lane / CH, n = group(a) == 1 ? row : att_div_g(a, row);
        return (uint32_t)n * (uint32_t)token(a) + (uint32_t)(row - n * group(a)) * (uint32_t)head(a) + (((lane % CH) ^ att_swz<DP>(row)) << 4);
    }
    __device__ __forceinline__ void init(const void* p, const AttArgs& a, int w, int lane) {
        const long long sn = token(a), sh = head(a);
        const int G = group(a);
        base = (const char*)p;
        step = sn * (ROWS / G);
        leap = NOFF == 1 ? sn * (LEAP / G) : 0;
        quick = a.D == DP && ROWS % G == 0 && (NOFF > 1 || LEAP % G == 0) && (unsigned long long)(step + sh * G) < 0x80000000ULL;
        if constexpr (HOLD)
#pragma unroll
            for (int i = 0; i < NOFF; ++i) off[i] = offset(a, i, w, lane);
    }
    // tile number `tile` of `rows` valid packed rows
    __device__ __forceinline__ void stage(int tile, int rows, char* lds, int w) const {
        if (quick && (tile + 1) * ROWS <= rows) {
            const char* b = base + tile * step;
            uint32_t once = 0;
            if constexpr (!HOLD) once = offset(*att_args(), 0, w, att_lane());
#pragma unroll
            for (int i = 0; i < N; ++i) dma_off(dma_base(b + i * leap), HOLD ? off[NOFF == 1 ? 0 : i] : once, lds + (i * NW + w) * 1024);
            return;
        }
        AttArgsMem& a = *att_args();
        const int lane = att_lane();
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
            const int lr = (i * NW + w) * RPP + lane / CH, row = tile * ROWS + lr;
            const int chunk = (lane % CH) ^ att_swz<DP>(lr);
            const int n = group(a) == 1 ? row : att_div_g(a, row);
            const char* p = base + n * token(a) + (row - n * group(a)) * head(a) + chunk * 16;
            dma_ptr(row < rows && chunk * 8 < a.D ? p : reinterpret_cast<const char*>(g_att_zero), lds + (i * NW + w) * 1024);
        }
    }
};

// A lane's place in a tile, for both kinds of fragment reads. The swizzle only flips bits 4 .. 7 of an address and repeats every 16 rows,
// so the slice (ks) and the channel block (db) are flips of the same bits: one register per kind, one exclusive-or per read.
template <int DP>
struct AttLane {
    int row, col;
    __device__ __forceinline__ AttLane(int lane) {
        const int r = lane & 31, h = lane >> 5;
        row = r * (DP * 2) + ((h ^ att_swz<DP>(r)) << 4);
        const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3, ra = 4 * (g >> 1) + q;
        col = ra * (DP * 2) + (((2 * (g & 1) + (p >> 1)) ^ att_swz<DP>(ra)) << 4) + 8 * (p & 1);
    }
    // in front of a loop body: keeps the flipped addresses of all slices from being computed outside and held there (16 registers)
    __device__ __forceinline__ void pin() { asm volatile("" : "+v"(row), "+v"(col)); }
};

// row fragment: lane (r, h) gets channels 16 ks + 8 h .. + 8 of tile row row0 + r (row0 % 16 == 0)
template <typename T, int DP>
__device__ __forceinline__ typename AttVec<T>::v8 att_row_frag(const char* lds, const AttLane<DP>& at, int row0, int ks) {
    return *reinterpret_cast<const typename AttVec<T>::v8*>(lds + row0 * (DP * 2) + (at.row ^ (ks << 5)));
}

// transposed fragment: lane (r, h) gets channel 32 db + r of tile rows row0 + 4h + {0..3} and row0 + 8 + 4h + {0..3} (row0 % 16 == 0;
// eight rows further the swizzle flips bit 5)
template <typename T, int DP>
__device__ __forceinline__ typename AttVec<T>::v8 att_col_frag(const char* lds, const AttLane<DP>& at, int row0, int db) {
    typedef typename AttVec<T>::v4 v4;
    const char* base = lds + row0 * (DP * 2);
    const v4 lo = ds_tr16((SVPS_LDS v4*)(base + (at.col ^ (db << 6))));
    const v4 hi = ds_tr16((SVPS_LDS v4*)(base + 8 * (DP * 2) + (at.col ^ 32 ^ (db << 6))));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// eight accumulator values to one operand fragment
template <typename T>
__device__ __forceinline__ typename AttVec<T>::v8 att_pack(const float* x) {
    typename AttVec<T>::v8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)x[j];
    return r;
}

// the reference point of a row that has seen no key: far below any score, finite, so that 2^(s - it) of a masked score is 0 and not NaN
constexpr float kAttFloor = -3.0e38f;

// a lane's 16 accumulator values of one 32-channel block (channels (i & 3) + 8 (i >> 2) + 4 h) of one row, times f, as 16-bit channels
template <typename T>
__device__ __forceinline__ void att_store_block(T* row, int d0, int h, int D, const f32x16& acc, float f) {
    typedef typename AttVec<T>::v4 v4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = d0 + 8 * g + 4 * h;
        if (d < D) {                                             // D % 8 == 0: a quad is inside or outside as a whole
            v4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = (T)(acc[4 * g + j] * f);
            *reinterpret_cast<v4*>(row + d) = o;
        }
    }
}

__device__ __forceinline__ void att_store_block_f32(float* row, int d0, int h, int D, const f32x16& acc) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = d0 + 8 * g + 4 * h;
        if (d < D) {
            f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = acc[4 * g + j];
            *reinterpret_cast<f32x4*>(row + d) = o;
        }
    }
}

}  // namespace svps
