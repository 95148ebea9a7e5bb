// relattn_backward.hip -- gradients of attention with a learned relative position bias for gfx950 (C-ABI: include/gvd_relattn.h).
//
//     P = exp2(S - lse),  dV = P^T dO,  dP = dO V^T,  dS = P o (dP - delta),  delta_i = sum_j P_ij dP_ij
//     dQ = scale dS K,  dK = scale dS^T Q,  dT[b, h] = sum of dS_ij over the (i, j) whose distance lies in bucket b
//
// General rows, kernels in turn, no sum whose order could change:
//   k_rel_dq      a wave = 32 queries; walks the keys with delta from dO . O.  O was rounded, and so were the P that made it, so this delta is up to 2^-8 |dO| |O| off
//                 (bf16), which is much where V has a mean (dS is a difference then) and for a table's gradient in 32 bits (its sums cancel: a row's dS
//                 sums to 0).  But a row's dS as formed sums to exactly what delta was off by, so dQ = dS K - (that sum) P K, one more product on K's
//                 fragments, and the delta that the kernel leaves for k_rel_dkv is right.  (V = noise + 3, bf16: dQ 2.1 % off without, 0.24 % with)
//   k_rel_dkv     a wave = 32 keys; walks the queries; dS of the table from the corrected delta: by distance into an array of the wave's own in LDS, blocks beyond
//                 the last border into one register; at the end distances are summed into buckets, one row of partial sums a workgroup
//   k_rel_table   sums the partial rows, 64 bits; an entry that masks or that counts as another value has no gradient
// P and dS are rounded to the inputs' 16 bits as operands of the second products, the only type the matrix unit takes at this rate: 2^-8 (bf16) or 2^-11 (fp16) of each at most, which sums of
// many terms average; the table is summed from dS in 32 bits.
// Bound by instruction issue (two waves a SIMD, 200 registers), and by the workgroups' number: 2304 rows, 10 heads, 180 workgroups on 256 CUs: 37 and 48 us in a loop of training passes, with
// or without a causal mask (a launch lasts as long as its longest walk); 9216 rows, 5 heads: 263 and 328 us, 830 and 660 TFLOP/s of 4 products each.
// Up to 32 queries and keys: k_rel_short_bwd, a wave an item as in the forward; the wave's head is fixed, so dS is summed over its items in registers and goes
// into buckets once.
#include "relattn_common.h"

using namespace gvdr;

namespace {

// Tiles of 64 rows x 64 channels in turn, through 512 lanes, 16 bytes each: eight lanes a row.  Rows at or behind n_rows: the last one again (n_rows >= 1).
// The address moves along: a row's number times the stride, in 64 bits, would take the vector unit as long as 40 additions a lane and tile.
template <typename T> struct TileRows {
    const T *at, *last;
    size_t step;
    int row, n_rows;

    __device__ __forceinline__ TileRows(const T* src, size_t rs, int row0, int n, int tid)
        : at(src + (size_t)(row0 + (tid >> 3)) * rs + (tid & 7) * 8), last(src + (size_t)(n > 0 ? n - 1 : 0) * rs + (tid & 7) * 8), step(64 * rs), row(row0 + (tid >> 3)), n_rows(n) {}
    __device__ __forceinline__ typename Tr<T>::vec8 next()
    {
        const auto x = *reinterpret_cast<const typename Tr<T>::vec8*>(row < n_rows ? at : last);
        at += step;
        row += 64;
        return x;
    }
};

template <typename T>
__device__ __forceinline__ void tile_commit(typename Tr<T>::vec8 x, int tid, T (*dst)[LDS_ROW])
{
    *reinterpret_cast<typename Tr<T>::vec8*>(&dst[tid >> 3][(tid & 7) * 8]) = x;
}

// 64 channels of one row from a C-layout pair (x0: channels 0 .. 31, x1: 32 .. 63)
template <typename T>
__device__ __forceinline__ void store_row(T* __restrict__ row, const f16v& x0, const f16v& x1, float mul, int hi)
{
#pragma unroll
    for (int rg = 0; rg < 4; rg++) {
        const int d0 = 8 * rg + 4 * hi;
        uint2 w;
        w.x = Tr<T>::pack2(x0[4 * rg] * mul, x0[4 * rg + 1] * mul);
        w.y = Tr<T>::pack2(x0[4 * rg + 2] * mul, x0[4 * rg + 3] * mul);
        *reinterpret_cast<uint2*>(row + d0) = w;
        w.x = Tr<T>::pack2(x1[4 * rg] * mul, x1[4 * rg + 1] * mul);
        w.y = Tr<T>::pack2(x1[4 * rg + 2] * mul, x1[4 * rg + 3] * mul);
        *reinterpret_cast<uint2*>(row + 32 + d0) = w;
    }
}

// Both kernels: 8 waves, two a SIMD.  Waves w and w + 4 share a block of 32 rows and take one half each of every 64-row tile of the other side; the second four hand
// their sums over through LDS at the end, in registers' order.  Tiles are double-buffered: one barrier a tile, loads two tiles ahead, also where those tiles lie
// behind the end: with branches around them, 2304 rows and 10 heads took 51 and 60 us instead of 48 and 57.  Rows at or behind the end come as the last one again and
// weigh 0 (the bias of -infinity they meet is set in registers; zeros in LDS instead: 3 us more).  Where in the loop the next tile's stores to LDS stand was measured,
// place by place: before the second products in k_rel_dq (43.8 us; first thing 45.3, last 49.7), last in k_rel_dkv (54.5; 55.6, 56.4 before the sums).
template <typename T> struct Tiles { T a[2][64][LDS_ROW], b[2][64][LDS_ROW]; };
constexpr int HANDOVER = 4 * 32 * 64 * (int)sizeof(float);   // 4 waves x 32 registers x 64 lanes: fits the tiles' LDS
static_assert(sizeof(Tiles<__bf16>) >= HANDOVER, "the hand-over uses the tiles' memory");

__device__ __forceinline__ void hand_over(float* at, int wave, int lane, const f16v& x0, const f16v& x1)
{
    float* p = at + (wave & 3) * 2048 + lane;
#pragma unroll
    for (int r = 0; r < 16; r++) { p[64 * r] = x0[r]; p[64 * (16 + r)] = x1[r]; }
}
__device__ __forceinline__ void take_over(const float* at, int wave, int lane, f16v& x0, f16v& x1)
{
    const float* p = at + (wave & 3) * 2048 + lane;
#pragma unroll
    for (int r = 0; r < 16; r++) { x0[r] += p[64 * r]; x1[r] += p[64 * (16 + r)]; }
}

// ---- dQ, and delta put right ---------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
k_rel_dq(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ o, const T* __restrict__ d_o,
         const float* __restrict__ lse, float* __restrict__ delta, T* __restrict__ dq)
{
    typedef typename Tr<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) Tiles<T> tiles;   // a: K, b: V
    __shared__ float sOff[8][32];
    extern __shared__ __attribute__((aligned(16))) float sBias[];

    int bh, tile_y;
    xcd_item_tile(bh, tile_y);
    const int b = bh / g.H, h = bh - b * g.H;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
    const int half = 32 * (wave >> 2);   // the half of each key tile
    const int start = start_of(g, b), len = len_of(g, b);
    const T* kb = k + (size_t)b * g.kv_bs + (size_t)h * 64;
    const T* vb = v + (size_t)b * g.kv_bs + (size_t)h * 64;
    const int q0 = tile_y * 128, query = q0 + (wave & 3) * 32 + col, q_last = (q0 + 128 < g.Nq ? q0 + 128 : g.Nq) - 1;
    const int first = start + q0 + (wave & 3) * 32;   // position of the wave's first query
    const int k_hi = g.causal ? clamp_int(start + q_last + 1, 0, len) : len;
    const int k_full = g.causal ? clamp_int(start + q0 + 1, 0, len) : len;
    const bool valid = query < g.Nq;
    const size_t qrow = (size_t)b * g.q_bs + (size_t)h * 64 + (size_t)(valid ? query : g.Nq - 1) * (size_t)g.q_rs;
    const size_t grow = (size_t)b * g.o_bs + (size_t)h * 64 + (size_t)(valid ? query : g.Nq - 1) * (size_t)g.o_rs;
    vec8 qf[4], gf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
        qf[ks] = *reinterpret_cast<const vec8*>(q + qrow + 16 * ks + 8 * hi);
        gf[ks] = *reinterpret_cast<const vec8*>(d_o + grow + 16 * ks + 8 * hi);
    }
    const float L = valid ? lse[(size_t)bh * g.Nq + query] : INFINITY;   // (infinite: every weight of the row is 0)
    if (L == INFINITY) {   // such a row has no gradient, whatever its dO holds: a NaN times a weight of 0 would not be 0
#pragma unroll
        for (int ks = 0; ks < 4; ks++) gf[ks] = vec8{};
    }
    float Dl = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
        const vec8 x = *reinterpret_cast<const vec8*>(o + grow + 16 * ks + 8 * hi);
#pragma unroll
        for (int j = 0; j < 8; j++) Dl = fmaf((float)x[j], (float)gf[ks][j], Dl);
    }
    Dl += __shfl_xor(Dl, 32, 64);
    f16v dq0 = {}, dq1 = {}, pk0 = {}, pk1 = {}, minus_delta;   // (dP's accumulators start from -delta: dS = P o what comes out)
#pragma unroll
    for (int r = 0; r < 16; r++) minus_delta[r] = -Dl;
    float off = 0.f;   // this lane's part of the row's sum of dS

    vec8 rk = {}, rv = {};
    TileRows<T> k_rows(kb, (size_t)g.kv_rs, 0, len, tid), v_rows(vb, (size_t)g.kv_rs, 0, len, tid);
    if (k_hi > 0) {
        rk = k_rows.next();
        rv = v_rows.next();
    }
    fill_bias(g, h, sBias, tid, 512);
    if (k_hi > 0) {
        tile_commit(rk, tid, tiles.a[0]);
        tile_commit(rv, tid, tiles.b[0]);
        rk = k_rows.next();
        rv = v_rows.next();
    }
    __syncthreads();
    const float far_past = sBias[0] * g.c, far_ahead = sBias[bias_len(g.reach) - 1] * g.c;
    int buf = 0;
    for (int kt = 0; kt < k_hi; kt += 64, buf ^= 1) {
        const int k0 = kt + half;   // the wave's 32 keys
        f16v s = {}, dp = minus_delta;
        float shift = -L;           // weights are exp2(s c + shift): a single bias of the block goes here
        const bool past = k0 + 31 - first <= -g.reach, ahead = k0 - first - 31 >= g.reach;
        if (past || ahead) shift += past ? far_past : far_ahead;
        else {
            const float* e = sBias + (k0 + 4 * hi - first - col + g.reach + PAD);
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = e[(r & 3) + 8 * (r >> 2)];
        }
#pragma unroll
        for (int ks = 0; ks < 4; ks++) s = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&tiles.a[buf][half + col][16 * ks + 8 * hi]), qf[ks], s);
        if (k0 + 32 > k_full) {
            const int seen = (g.causal && start + query + 1 < len ? start + query + 1 : len) - k0 - 4 * hi;
#pragma unroll
            for (int r = 0; r < 16; r++)
                if ((r & 3) + 8 * (r >> 2) >= seen) s[r] = -INFINITY;
        }
#pragma unroll
        for (int ks = 0; ks < 4; ks++) dp = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&tiles.b[buf][half + col][16 * ks + 8 * hi]), gf[ks], dp);
        unsigned pp[8], pd[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * j], g.c, shift)), p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], g.c, shift));
            const float d0 = p0 * dp[2 * j], d1 = p1 * dp[2 * j + 1];
            off += d0 + d1;
            pp[j] = Tr<T>::pack2(p0, p1);
            pd[j] = Tr<T>::pack2(d0, d1);
        }
        tile_commit(rk, tid, tiles.a[buf ^ 1]);
        tile_commit(rv, tid, tiles.b[buf ^ 1]);
        rk = k_rows.next();
        rv = v_rows.next();
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const vec8 df = packed_operand<T>(pd, k2), pf = packed_operand<T>(pp, k2);
            const vec8 a0 = transposed_operand(&tiles.a[buf][0][0], LDS_ROW, half + 16 * k2, 0, lane);
            const vec8 a1 = transposed_operand(&tiles.a[buf][0][0], LDS_ROW, half + 16 * k2, 32, lane);
            dq0 = Tr<T>::mfma(a0, df, dq0);
            dq1 = Tr<T>::mfma(a1, df, dq1);
            pk0 = Tr<T>::mfma(a0, pf, pk0);
            pk1 = Tr<T>::mfma(a1, pf, pk1);
        }
        __syncthreads();
    }
    off += __shfl_xor(off, 32, 64);
    if (hi == 0) sOff[wave][col] = off;
    __syncthreads();
    off = sOff[wave & 3][col] + sOff[(wave & 3) + 4][col];
#pragma unroll
    for (int r = 0; r < 16; r++) { dq0[r] = fmaf(-off, pk0[r], dq0[r]); dq1[r] = fmaf(-off, pk1[r], dq1[r]); }
    float* at = reinterpret_cast<float*>(&tiles);
    if (wave >= 4) hand_over(at, wave, lane, dq0, dq1);
    __syncthreads();
    if (wave < 4) {
        take_over(at, wave, lane, dq0, dq1);
        if (valid) {
            store_row<T>(dq + qrow, dq0, dq1, g.scale, hi);
            if (hi == 0) delta[(size_t)bh * g.Nq + query] = Dl + off;   // sum_j P dP = delta sum_j P + sum_j dS, and the weights sum to 1
        }
    }
}

// ---- dK, dV, and the table's partial sums ----------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
k_rel_dkv(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ d_o, const float* __restrict__ lse,
          const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part)
{
    typedef typename Tr<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) Tiles<T> tiles;   // a: Q, b: dO
    __shared__ __attribute__((aligned(16))) float sRow[2][2][64];   // -lse and -delta of a tile's rows
    __shared__ float sFar[8][2];
    __shared__ int sNone;   // whether some row may see nothing
    __shared__ float sSkew[8][16 * 48];
    extern __shared__ __attribute__((aligned(16))) float sBias[];   // the bias, then 8 arrays of sums by distance
    const int blen = bias_len(g.reach), span = g.reach + PAD;

    int bh, tile_y;
    xcd_item_tile(bh, tile_y);
    const int b = bh / g.H, h = bh - b * g.H;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
    const int half = 32 * (wave >> 2);   // the half of each query tile
    const int start = start_of(g, b), len = len_of(g, b);
    const T* qb = q + (size_t)b * g.q_bs + (size_t)h * 64;
    const T* gb = d_o + (size_t)b * g.o_bs + (size_t)h * 64;
    const size_t kvoff = (size_t)b * g.kv_bs + (size_t)h * 64;
    const float* row_b = (wave == 0 ? lse : delta) + (size_t)bh * g.Nq;   // what waves 0 and 1 bring

    const int k0 = tile_y * 128, kw = k0 + (wave & 3) * 32, key = kw + col;
    const bool there = key < len;
    float* sums = sBias + blen * (1 + wave);
    float* skew = &sSkew[wave][4 * hi * 47 + col + 15];   // element (row i, key col) of 16 rows: 48 i + col - i + 15
    const float* column = &sSkew[wave][lane < 47 ? lane : 47];
    vec8 kf[4], vf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
        const size_t kr = kvoff + (size_t)(key < g.Nk ? key : g.Nk - 1) * (size_t)g.kv_rs + 16 * ks + 8 * hi;
        kf[ks] = *reinterpret_cast<const vec8*>(k + kr);
        vf[ks] = *reinterpret_cast<const vec8*>(v + kr);
        if (!there) { kf[ks] = vec8{}; vf[ks] = vec8{}; }
    }
    f16v dk0 = {}, dk1 = {}, dv0 = {}, dv1 = {};
    float far_sum[2] = { 0.f, 0.f };   // dS of the blocks beyond the last border: past, ahead

    // queries that may see a key of this workgroup: all, or those at or behind its first key
    const int q_lo = k0 >= len ? g.Nq : (g.causal ? clamp_int(k0 - start, 0, g.Nq) / 64 * 64 : 0);
    vec8 rq = {}, rg = {};
    float rr = 0.f;
    TileRows<T> q_rows(qb, (size_t)g.q_rs, q_lo, g.Nq, tid), g_rows(gb, (size_t)g.o_rs, q_lo, g.Nq, tid);
    auto prefetch = [&](int qt) {   // (tiles in turn)
        rq = q_rows.next();
        rg = g_rows.next();
        if (wave < 2) rr = row_b[qt + lane < g.Nq ? qt + lane : g.Nq - 1];
    };
    auto commit = [&](int qt, int buf) {
        tile_commit(rq, tid, tiles.a[buf]);
        tile_commit(rg, tid, tiles.b[buf]);
        if (wave < 2) sRow[buf][wave][lane] = qt + lane < g.Nq ? -rr : (wave == 0 ? -INFINITY : 0.f);   // rows past the end weigh 0
    };
    if (q_lo < g.Nq) prefetch(q_lo);
    for (int e = tid; e < 8 * blen; e += 512) sBias[blen + e] = 0.f;
    for (int e = lane; e < 16 * 48; e += 64) sSkew[wave][e] = 0.f;
    // Rows that see nothing: those before the first key where causal, and where entries mask their buckets any row (a length of zero walks no queries).  Their weights are 0, and
    // their dO, whatever it holds, is put to 0 in LDS, tile by tile; where there can be none of them the loop pays one scalar branch.
    if (tid == 0) sNone = g.causal && start < 0;
    __syncthreads();
    if (fill_bias<true>(g, h, sBias, tid, 512)) sNone = 1;
    if (q_lo < g.Nq) {
        commit(q_lo, 0);
        prefetch(q_lo + 64);
    }
    __syncthreads();
    const float far_ahead = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sBias[0])));
    const float far_past = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sBias[blen - 1])));
    const bool none = __builtin_amdgcn_readfirstlane(sNone);
    // S starts from the bias; lse is subtracted behind the products, in the exponent: as a start it would be some 1 / c times larger than what is summed, and its
    // rounding steps with it (a table's gradient in 32 bits at 2304 rows: 1e-6 off, 7e-7 this way, where 32 bits throughout are 7e-7 off).
    int buf = 0;
    for (int qt = q_lo; qt < g.Nq; qt += 64, buf ^= 1) {
        if (none) {   // (the same for the whole workgroup)
            if (sRow[buf][0][tid >> 3] == -INFINITY) tile_commit(vec8{}, tid, tiles.b[buf]);
            __syncthreads();
        }
        const int first = start + qt + half;   // position of the block's first query
        const bool past = kw + 31 - first <= -g.reach, ahead = kw - first - 31 >= g.reach;
        f16v s, dp;
        f4v minus_lse[4];
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {   // rows 8 g4 + 4 hi + {0 .. 3}
            minus_lse[g4] = *reinterpret_cast<const f4v*>(&sRow[buf][0][half + 8 * g4 + 4 * hi]);
            const f4v D = *reinterpret_cast<const f4v*>(&sRow[buf][1][half + 8 * g4 + 4 * hi]);
#pragma unroll
            for (int j = 0; j < 4; j++) dp[4 * g4 + j] = D[j];
        }
        if (past || ahead) {
            const float far = past ? far_past : far_ahead;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = far;
        } else {
            const float* e = sBias + (first + 4 * hi - key + span);   // (descending distances: row r at + (r & 3) + 8 (r >> 2))
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = e[(r & 3) + 8 * (r >> 2)];
        }
#pragma unroll
        for (int ks = 0; ks < 4; ks++) s = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&tiles.a[buf][half + col][16 * ks + 8 * hi]), kf[ks], s);
        if (kw + 32 > len || (g.causal && kw + 31 > first)) {
            const int least = !there ? 0x7fffffff : (g.causal ? key - first - 4 * hi : -64);   // the key's first row that sees it
#pragma unroll
            for (int r = 0; r < 16; r++)
                if ((r & 3) + 8 * (r >> 2) < least) s[r] = -INFINITY;
        }
#pragma unroll
        for (int ks = 0; ks < 4; ks++) dp = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&tiles.b[buf][half + col][16 * ks + 8 * hi]), vf[ks], dp);
        float ds[16];
        unsigned pp[8], pd[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const f4v L = minus_lse[j >> 1];
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * j], g.c, L[2 * (j & 1)])), p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], g.c, L[2 * (j & 1) + 1]));
            ds[2 * j] = p0 * dp[2 * j];
            ds[2 * j + 1] = p1 * dp[2 * j + 1];
            pp[j] = Tr<T>::pack2(p0, p1);
            pd[j] = Tr<T>::pack2(ds[2 * j], ds[2 * j + 1]);
        }
        if (past || ahead) {
            float x = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) x += ds[r];
            if (past) far_sum[0] += x; else far_sum[1] += x;
        } else {
            // by distance: 16 rows at a time go into the wave's own rows of LDS, each shifted by its number, so that a distance is a column; a lane sums a column.
            // (What a row leaves uncovered was zeroed once.  One addition in LDS an element instead: 6 us a tile, against 1.5 for all else.)
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (int r = 0; r < 8; r++) skew[((r & 3) + 8 * (r >> 2)) * 47] = ds[8 * x + r];
                wave_order();
                float y = 0.f, z = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r += 2) { y += column[48 * r]; z += column[48 * (r + 1)]; }
                if (lane < 47) sums[kw - first - 16 * x + lane - 15 + span] += y + z;
                wave_order();
            }
        }
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const vec8 pf = packed_operand<T>(pp, k2), df = packed_operand<T>(pd, k2);
            dv0 = Tr<T>::mfma(transposed_operand(&tiles.b[buf][0][0], LDS_ROW, half + 16 * k2, 0, lane), pf, dv0);
            dv1 = Tr<T>::mfma(transposed_operand(&tiles.b[buf][0][0], LDS_ROW, half + 16 * k2, 32, lane), pf, dv1);
            dk0 = Tr<T>::mfma(transposed_operand(&tiles.a[buf][0][0], LDS_ROW, half + 16 * k2, 0, lane), df, dk0);
            dk1 = Tr<T>::mfma(transposed_operand(&tiles.a[buf][0][0], LDS_ROW, half + 16 * k2, 32, lane), df, dk1);
        }
        commit(qt + 64, buf ^ 1);
        prefetch(qt + 128);
        __syncthreads();
    }
    float* at = reinterpret_cast<float*>(&tiles);
    if (wave >= 4) hand_over(at, wave, lane, dk0, dk1);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float x = far_sum[i];
#pragma unroll
        for (int w = 32; w; w >>= 1) x += __shfl_xor(x, w, 64);
        if (lane == 0) sFar[wave][i] = x;
    }
    __syncthreads();
    if (wave < 4) {
        take_over(at, wave, lane, dk0, dk1);
        if (key < g.Nk) store_row<T>(dk + kvoff + (size_t)key * (size_t)g.kv_rs, dk0, dk1, g.scale, hi);   // (behind the length: zeros)
    }
    __syncthreads();
    if (wave >= 4) hand_over(at, wave, lane, dv0, dv1);
    // distances into buckets
    for (int e = tid; e < blen; e += 512) {
        float x = 0.f;
#pragma unroll
        for (int w = 1; w <= 8; w++) x += sBias[w * blen + e];
        sBias[e] = x;
    }
    __syncthreads();
    if (wave < 4) {
        take_over(at, wave, lane, dv0, dv1);
        if (key < g.Nk) store_row<T>(dv + kvoff + (size_t)key * (size_t)g.kv_rs, dv0, dv1, 1.0f, hi);
    }
    float past = 0.f, ahead = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) { past += sFar[w][0]; ahead += sFar[w][1]; }
    const int l16 = tid & 15;
    for (int bucket = tid >> 4; bucket < g.buckets; bucket += 32) {   // 16 lanes a bucket
        const bool fore = bucket >= g.side;
        const int n_ = fore ? bucket - g.side : bucket;   // the bucket within its direction: distances lo .. up of it
        const int lo = g.first[n_], up = n_ + 1 < g.side ? g.first[n_ + 1] - 1 : span;
        float x = 0.f;
        for (int n = lo + l16; n <= up; n += 16)
            if (!fore || n > 0) x += sBias[fore ? span + n : span - n];
        if (!g.both && bucket == 0)   // one direction: whatever lies ahead shares the bucket of distance 0
            for (int n = 1 + l16; n <= span; n += 16) x += sBias[span + n];
#pragma unroll
        for (int w = 8; w; w >>= 1) x += __shfl_xor(x, w, 16);
        if (bucket == g.side - 1) x += past;
        if (bucket == (g.both ? g.buckets - 1 : 0)) x += ahead;
        if (l16 == 0) part[((size_t)bh * gridDim.y + tile_y) * g.buckets + bucket] = x;
    }
}

// Partial rows j = 0 .. count - 1 of head h lie at row ((j / tiles) H + h) tiles + j % tiles.  A wave a table entry, 64 bits, fixed order.
template <typename E>
__global__ void __launch_bounds__(64) k_rel_table(const float* __restrict__ part, const E* __restrict__ table, E* __restrict__ dtable, int H, int buckets, int tiles, int count)
{
    const int bucket = blockIdx.x, h = blockIdx.y;
    double x = 0.0;
    for (int j0 = threadIdx.x; j0 < count; j0 += 512) {   // eight loads in flight
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = j0 + 64 * i;
            y[i] = j < count ? part[(((size_t)(j / tiles) * H + h) * tiles + j % tiles) * buckets + bucket] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x += (double)y[i];
    }
#pragma unroll
    for (int w = 32; w; w >>= 1) x += __shfl_xor(x, w, 64);
    if (threadIdx.x == 0) dtable[bucket * H + h] = without_gradient((float)table[bucket * H + h]) ? (E)0.f : (E)(float)x;
}

// ---- up to 32 queries and keys -------------------------------------------------------------------------------------------------
// Both orientations of the score block are computed (a query per lane for dQ, delta and the table; a key per lane for dK and dV): 16 small products instead of a
// transposition of the weights; delta = sum_j P dP directly, O is not read.  Rows are read whole, 8 lanes each, and lie in LDS, where all operand forms come from;
// V's place takes the results on their way out.  The next item's rows are requested as soon as this one's lie there.
template <typename T>
__global__ void __launch_bounds__(256, 2) k_rel_short_bwd(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ d_o,
                                                          const float* __restrict__ lse, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv,
                                                          float* __restrict__ part, int items, int waves)
{
    typedef typename Tr<T>::vec8 vec8;
    constexpr int OP = 72;
    __shared__ __attribute__((aligned(16))) T sQ[4][32][OP];
    __shared__ __attribute__((aligned(16))) T sK[4][32][OP];
    __shared__ __attribute__((aligned(16))) T sG[4][32][OP];
    __shared__ __attribute__((aligned(16))) T sV[4][32][OP];
    __shared__ __attribute__((aligned(16))) float sL[4][32];
    __shared__ __attribute__((aligned(16))) float sD[4][32];
    __shared__ float sB[4][64];   // (75776 bytes in all: two workgroups a CU)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, r32 = lane & 31;
    const int gw = blockIdx.x * 4 + wave;
    if (gw >= waves) return;   // (no barriers below)
    const int h = gw % g.H, step = waves / g.H, nb = items / g.H, start = start_of(g, 0);
    const int row = lane >> 3, c8 = 8 * (lane & 7);   // rows 8 i + row
    sB[wave][lane] = start_value(g, table_at(g, bucket_of(g, lane - 32 - start), h));   // distances -32 .. 31 less the start
    wave_order();
    const float* bias_q = &sB[wave][4 * hi - r32 + 32];        // key row r: + (r & 3) + 8 (r >> 2)
    const float* bias_k = &sB[wave][r32 - 4 * hi + 32 - 27];   // query row r: + 27 - (r & 3) - 8 (r >> 2)
    f16v acc = {};   // dS^T summed over the wave's items

    vec8 rq[4], rk[4], rv[4], rg[4];
    float L_next;
    int len_next;
    auto load_kv = [&](int b) {
        int row_ = row;
        asm volatile("" : "+v"(row_));   // (not kept from item to item: the registers are full)
        len_next = len_of(g, b);
        const int last = len_next > 0 ? len_next - 1 : 0;
        const size_t kv = (size_t)b * g.kv_bs + (size_t)h * 64 + c8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + row_;
            const size_t j = r < last ? r : last;
            rk[i] = *reinterpret_cast<const vec8*>(k + kv + j * (size_t)g.kv_rs);
            rv[i] = *reinterpret_cast<const vec8*>(v + kv + j * (size_t)g.kv_rs);
        }
    };
    auto load_q = [&](int b) {
        int row_ = row;
        asm volatile("" : "+v"(row_));   // (not kept from item to item: the registers are full)
        const size_t qb = (size_t)b * g.q_bs + (size_t)h * 64 + c8, gb = (size_t)b * g.o_bs + (size_t)h * 64 + c8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + row_;
            const size_t n = r < g.Nq ? r : g.Nq - 1;
            rq[i] = *reinterpret_cast<const vec8*>(q + qb + n * (size_t)g.q_rs);
            rg[i] = *reinterpret_cast<const vec8*>(d_o + gb + n * (size_t)g.o_rs);
        }
        L_next = lse[((size_t)b * g.H + h) * g.Nq + (r32 < g.Nq ? r32 : g.Nq - 1)];
    };
    auto operand = [&](const T (&x)[32][OP], int ks) { return *reinterpret_cast<const vec8*>(&x[r32][16 * ks + 8 * hi]); };
    auto store_rows = [&](const f16v& x0, const f16v& x1, float mul, T* base, size_t rstride, int nrows) {
        int row_ = row;
        asm volatile("" : "+v"(row_));   // (not kept from item to item: the registers are full)
        store_row<T>(&sV[wave][r32][0], x0, x1, mul, hi);
        wave_order();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + row_;
            const u4 w = *reinterpret_cast<const u4*>(&sV[wave][r][c8]);
            if (r < nrows) __builtin_nontemporal_store(w, reinterpret_cast<u4*>(base + (size_t)r * rstride + c8));
        }
        wave_order();
    };

    load_kv(gw / g.H);
    load_q(gw / g.H);
    for (int b = gw / g.H; b < nb; b += step) {
        const int len = len_next;
        const size_t qbase = (size_t)b * g.q_bs + (size_t)h * 64, kbase = (size_t)b * g.kv_bs + (size_t)h * 64;
        const float L = r32 < g.Nq ? L_next : INFINITY;   // (rows past the end weigh 0)
        if (len == 0) {   // row 0 was loaded, whatever it holds: a NaN times a weight of 0 would not be 0
#pragma unroll
            for (int i = 0; i < 4; i++) { rk[i] = vec8{}; rv[i] = vec8{}; }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            *reinterpret_cast<vec8*>(&sK[wave][8 * i + row][c8]) = rk[i];
            *reinterpret_cast<vec8*>(&sQ[wave][8 * i + row][c8]) = rq[i];
            *reinterpret_cast<vec8*>(&sV[wave][8 * i + row][c8]) = rv[i];
            *reinterpret_cast<vec8*>(&sG[wave][8 * i + row][c8]) = rg[i];
        }
        load_kv(b + step < nb ? b + step : b);   // in flight under everything below
        wave_order();
        if (__any(L == INFINITY && r32 < g.Nq)) {   // rows that see nothing have no gradient, whatever their dO (and, with a length of zero, their query) holds
            if (L == INFINITY)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    *reinterpret_cast<vec8*>(&sG[wave][r32][32 * hi + 8 * i]) = vec8{};
                    if (len == 0) *reinterpret_cast<vec8*>(&sQ[wave][r32][32 * hi + 8 * i]) = vec8{};
                }
            wave_order();
        }
        // ---- a query per lane ----
        f16v sT, dpT = {};
#pragma unroll
        for (int r = 0; r < 16; r++) sT[r] = bias_q[(r & 3) + 8 * (r >> 2)];
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            sT = Tr<T>::mfma(operand(sK[wave], ks), operand(sQ[wave], ks), sT);
            dpT = Tr<T>::mfma(operand(sV[wave], ks), operand(sG[wave], ks), dpT);
        }
        const int seen = (g.causal && start + r32 + 1 < len ? start + r32 + 1 : len) - 4 * hi;
        float p[16], dl = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            p[r] = (r & 3) + 8 * (r >> 2) >= seen ? 0.f : __builtin_amdgcn_exp2f(fmaf(sT[r], g.c, -L));
            dl = fmaf(p[r], dpT[r], dl);
        }
        dl += __shfl_xor(dl, 32, 64);
        unsigned pdT[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d0 = p[2 * j] * (dpT[2 * j] - dl), d1 = p[2 * j + 1] * (dpT[2 * j + 1] - dl);
            acc[2 * j] += d0;
            acc[2 * j + 1] += d1;
            pdT[j] = Tr<T>::pack2(d0, d1);
        }
        if (hi == 0) {
            sL[wave][r32] = L;
            sD[wave][r32] = dl;
        }
        wave_order();
        f16v a0 = {}, a1 = {};
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const vec8 df = packed_operand<T>(pdT, k2);
            a0 = Tr<T>::mfma(transposed_operand(&sK[wave][0][0], OP, 16 * k2, 0, lane), df, a0);
            a1 = Tr<T>::mfma(transposed_operand(&sK[wave][0][0], OP, 16 * k2, 32, lane), df, a1);
        }
        // ---- a key per lane ----
        f16v s, dp = {};
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = bias_k[27 - (r & 3) - 8 * (r >> 2)];
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            s = Tr<T>::mfma(operand(sQ[wave], ks), operand(sK[wave], ks), s);
            dp = Tr<T>::mfma(operand(sG[wave], ks), operand(sV[wave], ks), dp);
        }
        load_q(b + step < nb ? b + step : b);
        wave_order();
        store_rows(a0, a1, g.scale, dq + qbase, (size_t)g.q_rs, g.Nq);
        const int least = r32 >= len ? 64 : (g.causal ? r32 - start - 4 * hi : -64);   // the first query row that sees this lane's key
        unsigned pp[8], pd[8];
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
            const float4 L4 = *reinterpret_cast<const float4*>(&sL[wave][8 * g4 + 4 * hi]);
            const float4 D4 = *reinterpret_cast<const float4*>(&sD[wave][8 * g4 + 4 * hi]);
            const float p0 = 8 * g4 + 0 < least ? 0.f : __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 0], g.c, -L4.x));
            const float p1 = 8 * g4 + 1 < least ? 0.f : __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 1], g.c, -L4.y));
            const float p2 = 8 * g4 + 2 < least ? 0.f : __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 2], g.c, -L4.z));
            const float p3 = 8 * g4 + 3 < least ? 0.f : __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 3], g.c, -L4.w));
            pp[2 * g4] = Tr<T>::pack2(p0, p1);
            pp[2 * g4 + 1] = Tr<T>::pack2(p2, p3);
            pd[2 * g4] = Tr<T>::pack2(p0 * (dp[4 * g4 + 0] - D4.x), p1 * (dp[4 * g4 + 1] - D4.y));
            pd[2 * g4 + 1] = Tr<T>::pack2(p2 * (dp[4 * g4 + 2] - D4.z), p3 * (dp[4 * g4 + 3] - D4.w));
        }
        f16v dv0 = {}, dv1 = {}, dk0 = {}, dk1 = {};
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const vec8 pf = packed_operand<T>(pp, k2), df = packed_operand<T>(pd, k2);
            dv0 = Tr<T>::mfma(transposed_operand(&sG[wave][0][0], OP, 16 * k2, 0, lane), pf, dv0);
            dv1 = Tr<T>::mfma(transposed_operand(&sG[wave][0][0], OP, 16 * k2, 32, lane), pf, dv1);
            dk0 = Tr<T>::mfma(transposed_operand(&sQ[wave][0][0], OP, 16 * k2, 0, lane), df, dk0);
            dk1 = Tr<T>::mfma(transposed_operand(&sQ[wave][0][0], OP, 16 * k2, 32, lane), df, dk1);
        }
        store_rows(dv0, dv1, 1.0f, dv + kbase, (size_t)g.kv_rs, g.Nk);
        store_rows(dk0, dk1, g.scale, dk + kbase, (size_t)g.kv_rs, g.Nk);
    }
    // dS^T by distance (a lane each: 31 at most on either side), then by bucket
    float* block = reinterpret_cast<float*>(&sV[wave][0][0]);   // [32 keys][33], then 64 buckets: 4480 of the wave's 4608 bytes
#pragma unroll
    for (int r = 0; r < 16; r++) block[((r & 3) + 8 * (r >> 2) + 4 * hi) * 33 + r32] = acc[r];
    wave_order();
    float x = 0.f;
    for (int i = 0; i < 32; i++) {
        const int j = i + lane - 32;
        if (j >= 0 && j < 32) x += block[j * 33 + i];
    }
    int* sBk = reinterpret_cast<int*>(block + 32 * 33);
    sB[wave][lane] = x;
    sBk[lane] = bucket_of(g, lane - 32 - start);
    wave_order();
    for (int bucket = lane; bucket < g.buckets; bucket += 64) {
        float y = 0.f;
        for (int e = 0; e < 64; e++) y += sBk[e] == bucket ? sB[wave][e] : 0.f;
        part[(size_t)gw * g.buckets + bucket] = y;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
bool is_short(const Geo& g) { return g.Nq <= 32 && g.Nk <= 32; }

// waves of the short form: what stays resident (LDS and registers: two workgroups of 4 a CU), a multiple of the heads
int short_waves(const Geo& g, int B)
{
    long long waves = (long long)compute_units() * 8;
    if (waves > (long long)B * g.H) waves = (long long)B * g.H;
    return (int)(waves >= g.H ? waves / g.H * g.H : g.H);
}

long long partial_rows(const Geo& g, int B) { return is_short(g) ? short_waves(g, B) : (long long)B * g.H * ((g.Nk + 127) / 128); }

template <typename T>
int launch_bwd(const Geo& g, int B, const void* q, const void* k, const void* v, const void* out, const void* d_o, const float* lse, void* dq, void* dk, void* dv,
               void* dtable, float* ws, hipStream_t stream)
{
    const int BH = B * g.H;
    float* part = ws;
    float* delta = ws + partial_rows(g, B) * g.buckets;
    int tiles, count;
    if (is_short(g)) {
        const int waves = short_waves(g, B);
        tiles = 1;
        count = waves / g.H;
        hipLaunchKernelGGL(k_rel_short_bwd<T>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream, g, (const T*)q, (const T*)k, (const T*)v, (const T*)d_o, lse,
                           (T*)dq, (T*)dk, (T*)dv, part, BH, waves);
    } else {
        tiles = (g.Nk + 127) / 128;
        const int qtiles = (g.Nq + 127) / 128;
        if (BH > (1 << 22) || tiles > 65535 || qtiles > 65535 || (long long)BH * (tiles > qtiles ? tiles : qtiles) > 0x7fffffffLL)
            return fail(-1, "gvd_relattn_bwd: too many workgroups");
        count = B * tiles;
        const size_t lds = sizeof(float) * bias_len(g.reach);
        hipLaunchKernelGGL(k_rel_dq<T>, dim3((unsigned)BH, (unsigned)qtiles), dim3(512), lds, stream, g, (const T*)q, (const T*)k, (const T*)v, (const T*)out,
                           (const T*)d_o, lse, delta, (T*)dq);
        hipLaunchKernelGGL(k_rel_dkv<T>, dim3((unsigned)BH, (unsigned)tiles), dim3(512), 9 * lds, stream, g, (const T*)q, (const T*)k, (const T*)v, (const T*)d_o, lse,
                           (const float*)delta, (T*)dk, (T*)dv, part);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(-2, "launch k_rel_*_bwd", e);
    const dim3 grid((unsigned)g.buckets, (unsigned)g.H);
#define GVD_TABLE(E) hipLaunchKernelGGL(k_rel_table<E>, grid, dim3(64), 0, stream, (const float*)part, (const E*)g.table, (E*)dtable, g.H, g.buckets, tiles, count)
    if (g.table_type == 0) GVD_TABLE(float); else if (g.table_type == 1) GVD_TABLE(_Float16); else GVD_TABLE(__bf16);
#undef GVD_TABLE
    e = hipGetLastError();
    if (e != hipSuccess) return fail(-2, "launch k_rel_table", e);
    return 0;
}

}  // namespace

extern "C" {

long long gvd_relattn_bwd_workspace(const gvd_relattn_problem* p)
{
    Geo g;
    const int rc = make_geo(p, g, "gvd_relattn_bwd_workspace");
    if (rc) return rc;
    return (long long)sizeof(float) * (partial_rows(g, p->B) * g.buckets + (is_short(g) ? 0 : (long long)p->B * p->H * p->Nq));
}

int gvd_relattn_bwd(const gvd_relattn_problem* p, const void* q, const void* k, const void* v, const void* table, const void* out, const void* d_out,
                    const float* lse, void* dq, void* dk, void* dv, void* dtable, void* workspace, void* stream)
{
    Geo g;
    const int rc = make_geo(p, g, "gvd_relattn_bwd");
    if (rc) return rc;
    if (p->q_starts) return fail(-1, "gvd_relattn_bwd: one q_start for the whole batch only");
    if (p->kv_bs == 0 && p->B > 1) return fail(-1, "gvd_relattn_bwd: keys and values shared by the batch have no gradient here");
    if (p->H > 65535) return fail(-1, "gvd_relattn_bwd: too many heads");
    if (!q || !k || !v || !table || !out || !d_out || !lse || !dq || !dk || !dv || !dtable || !workspace) return fail(-1, "gvd_relattn_bwd: null pointer");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)d_out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15)
        return fail(-1, "gvd_relattn_bwd: pointers must be 16-byte aligned");
    g.table = table;
    return p->is_bf16 ? launch_bwd<__bf16>(g, p->B, q, k, v, out, d_out, lse, dq, dk, dv, dtable, (float*)workspace, (hipStream_t)stream)
                      : launch_bwd<_Float16>(g, p->B, q, k, v, out, d_out, lse, dq, dk, dv, dtable, (float*)workspace, (hipStream_t)stream);
}

}  // extern "C"
