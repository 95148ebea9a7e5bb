// relattn_backward.hip -- gradients of attention with a learned relative position bias for gfx950 (C-ABI: include/gvd_relattn.h).
//
//     P = exp2(S - lse),  dV = P^T dO,  dP = dO V^T,  dS = P o (dP - delta),  delta_i = sum_j P_ij dP_ij
//     dQ = scale dS K,  dK = scale dS^T Q,  dT[b, h] = sum of dS_ij over the (i, j) whose distance lies in bucket b
//
// General rows, three kernels in turn, no sum whose order could change:
//   k_rel_delta   delta from dO . O: O was rounded, and so were the P that made it, so this delta is 2^-9 off (bf16) -- enough for 16-bit gradients, not for
//                 a table's gradient in 32 bits: its sums cancel (a row's dS sums to 0)
//   k_rel_dq      a wave = 32 queries; walks the keys; also sums each row's dS, which is exactly what delta was off by, and puts delta right
//   k_rel_dkv     a wave = 32 keys; walks the queries; dS of the table from the corrected delta: by distance into an array of the wave's own in LDS (a 32 x 32 block
//                 adds its rows one half wave at a time: all lanes at different distances), blocks beyond the last border into one register; at the end
//                 distances are summed into buckets, one row of partial sums a workgroup
//   k_rel_table   sums the partial rows, 64 bits
// Up to 32 queries and keys: k_rel_short_bwd, a wave an item as in the forward; the wave's head is fixed, so dS is summed over its items in registers and goes
// into buckets once.
#include "relattn_common.h"

using namespace gvdr;

namespace {

template <typename T>
__global__ void __launch_bounds__(256) k_rel_delta(const Geo g, const T* __restrict__ o, const T* __restrict__ d_o, float* __restrict__ delta, long long rows)
{
    typedef typename Tr<T>::vec8 vec8;
    const long long i = (long long)blockIdx.x * 32 + (threadIdx.x >> 3);   // (b H + h) Nq + n; 8 lanes a row
    if (i >= rows) return;
    const long long bh = i / g.Nq;
    const int n = (int)(i - bh * g.Nq), b = (int)(bh / g.H), h = (int)(bh - (long long)b * g.H);
    const size_t off = (size_t)b * g.o_bs + (size_t)n * g.o_rs + (size_t)h * 64 + 8 * (threadIdx.x & 7);
    const vec8 x = *reinterpret_cast<const vec8*>(o + off), y = *reinterpret_cast<const vec8*>(d_o + off);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) s = fmaf((float)x[j], (float)y[j], s);
    s += __shfl_xor(s, 1, 64);
    s += __shfl_xor(s, 2, 64);
    s += __shfl_xor(s, 4, 64);
    if ((threadIdx.x & 7) == 0) delta[i] = s;
}

// A tile of 64 rows x 64 channels: registers, then LDS row-major and (TRANSPOSED) channel-major with two rows a dword.  Loads are unconditional (the last valid row
// again; n_rows >= 1) and committed as zeros beyond n_rows.
template <typename T> struct TileRegs { typename Tr<T>::vec8 r[2], t0, t1; };

template <typename T, bool TRANSPOSED>
__device__ __forceinline__ void tile_load(const T* __restrict__ src, size_t rs, int row0, int n_rows, int tid, TileRegs<T>& R)
{
    typedef typename Tr<T>::vec8 vec8;
    const int last = n_rows - 1;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int c = tid + i * 256, g = row0 + (c >> 3);
        R.r[i] = *reinterpret_cast<const vec8*>(src + (size_t)(g < last ? g : last) * rs + (c & 7) * 8);
    }
    if (TRANSPOSED) {
        const int g = row0 + 2 * (tid & 31), c8 = (tid >> 5) * 8;
        R.t0 = *reinterpret_cast<const vec8*>(src + (size_t)(g < last ? g : last) * rs + c8);
        R.t1 = *reinterpret_cast<const vec8*>(src + (size_t)(g + 1 < last ? g + 1 : last) * rs + c8);
    }
}

template <typename T, bool TRANSPOSED>
__device__ __forceinline__ void tile_commit(int row0, int n_rows, int tid, const TileRegs<T>& R, T (*sRow)[LDS_ROW], T (*sTr)[LDS_ROW])
{
    typedef typename Tr<T>::vec8 vec8;
    typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int c = tid + i * 256, row = c >> 3;
        *reinterpret_cast<vec8*>(&sRow[row][(c & 7) * 8]) = (row0 + row < n_rows) ? R.r[i] : vec8{};
    }
    if (TRANSPOSED) {
        const int kp = tid & 31, c8 = (tid >> 5) * 8, g = row0 + 2 * kp;
        const vec8 x0 = (g < n_rows) ? R.t0 : vec8{}, x1 = (g + 1 < n_rows) ? R.t1 : vec8{};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const T2 pr = { x0[i], x1[i] };
            *reinterpret_cast<T2*>(&sTr[c8 + i][2 * kp]) = pr;
        }
    }
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

// ---- dQ, and delta put right ---------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
k_rel_dq(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ d_o, const float* __restrict__ lse,
         float* __restrict__ delta, T* __restrict__ dq)
{
    typedef typename Tr<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) T sK[64][LDS_ROW];
    __shared__ __attribute__((aligned(16))) T sV[64][LDS_ROW];
    __shared__ __attribute__((aligned(16))) T sKt[64][LDS_ROW];
    extern __shared__ __attribute__((aligned(16))) float sBias[];

    int bh, tile_y;
    xcd_item_tile(bh, tile_y);
    const int b = bh / g.H, h = bh - b * g.H;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
    const int start = start_of(g, b), len = len_of(g, b);
    const T* kb = k + (size_t)b * g.kv_bs + (size_t)h * 64;
    const T* vb = v + (size_t)b * g.kv_bs + (size_t)h * 64;
    const int q0 = tile_y * 128, query = q0 + wave * 32 + col, q_last = (q0 + 128 < g.Nq ? q0 + 128 : g.Nq) - 1;
    const int first = start + q0 + wave * 32;   // position of the wave's first query
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
    const float Dl = valid ? delta[(size_t)bh * g.Nq + query] : 0.f;
    f16v dq0 = {}, dq1 = {};
    float off = 0.f;   // this lane's part of the row's sum of dS

    TileRegs<T> rk, rv;
    if (k_hi > 0) {
        tile_load<T, true>(kb, (size_t)g.kv_rs, 0, len, tid, rk);
        tile_load<T, false>(vb, (size_t)g.kv_rs, 0, len, tid, rv);
    }
    fill_bias(g, h, sBias, tid, 256);
    __syncthreads();
    const float far_past = sBias[0], far_ahead = sBias[bias_len(g.reach) - 1];
    for (int kt = 0; kt < k_hi; kt += 64) {
        __syncthreads();
        tile_commit<T, true>(kt, len, tid, rk, sK, sKt);
        tile_commit<T, false>(kt, len, tid, rv, sV, nullptr);
        if (kt + 64 < k_hi) {
            tile_load<T, true>(kb, (size_t)g.kv_rs, kt + 64, len, tid, rk);
            tile_load<T, false>(vb, (size_t)g.kv_rs, kt + 64, len, tid, rv);
        }
        __syncthreads();
        const bool masked = kt + 64 > k_full;
        const bool far = kt + 63 - first <= -g.reach || kt - first - 31 >= g.reach;
#pragma unroll
        for (int kbk = 0; kbk < 2; kbk++) {
            f16v s, dp = {};
            if (far) {
                const float x = kt < first ? far_past : far_ahead;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = x;
            } else {
                const float* e = sBias + (kt + 32 * kbk + 4 * hi - first - col + g.reach + PAD);
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = e[(r & 3) + 8 * (r >> 2)];
            }
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                const vec8 ak = *reinterpret_cast<const vec8*>(&sK[32 * kbk + col][16 * ks + 8 * hi]);
                const vec8 av = *reinterpret_cast<const vec8*>(&sV[32 * kbk + col][16 * ks + 8 * hi]);
                s = Tr<T>::mfma(ak, qf[ks], s);
                dp = Tr<T>::mfma(av, gf[ks], dp);
            }
            if (masked) {
                const int seen = (g.causal && start + query + 1 < len ? start + query + 1 : len) - kt - 32 * kbk - 4 * hi;
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if ((r & 3) + 8 * (r >> 2) >= seen) s[r] = -INFINITY;
            }
            unsigned pd[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float d0 = __builtin_amdgcn_exp2f(fmaf(s[2 * j], g.c, -L)) * (dp[2 * j] - Dl);
                const float d1 = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], g.c, -L)) * (dp[2 * j + 1] - Dl);
                off += d0 + d1;
                pd[j] = Tr<T>::pack2(d0, d1);
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; k2++) {
                const vec8 df = packed_c_to_b_operand<T>(pd, k2);
                const int kc = 32 * kbk + 16 * k2 + 8 * hi;
                dq0 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sKt[col][kc]), df, dq0);
                dq1 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sKt[32 + col][kc]), df, dq1);
            }
        }
    }
    off += __shfl_xor(off, 32, 64);
    if (valid) {
        store_row<T>(dq + qrow, dq0, dq1, g.scale, hi);
        if (hi == 0) delta[(size_t)bh * g.Nq + query] = Dl + off;   // sum_j P dP = delta sum_j P + sum_j dS, and the weights sum to 1
    }
}

// ---- dK, dV, and the table's partial sums ----------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
k_rel_dkv(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ d_o, const float* __restrict__ lse,
          const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part)
{
    typedef typename Tr<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) T sQ[64][LDS_ROW];
    __shared__ __attribute__((aligned(16))) T sdO[64][LDS_ROW];
    __shared__ __attribute__((aligned(16))) T sQt[64][LDS_ROW];
    __shared__ __attribute__((aligned(16))) T sdOt[64][LDS_ROW];
    __shared__ __attribute__((aligned(16))) float sLse[64];
    __shared__ __attribute__((aligned(16))) float sDelta[64];
    __shared__ float sFar[4][2];
    extern __shared__ __attribute__((aligned(16))) float sBias[];   // the bias, then 4 arrays of sums by distance
    const int blen = bias_len(g.reach), span = g.reach + PAD;

    int bh, tile_y;
    xcd_item_tile(bh, tile_y);
    const int b = bh / g.H, h = bh - b * g.H;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, col = lane & 31;
    const int start = start_of(g, b), len = len_of(g, b);
    const T* qb = q + (size_t)b * g.q_bs + (size_t)h * 64;
    const T* gb = d_o + (size_t)b * g.o_bs + (size_t)h * 64;
    const size_t kvoff = (size_t)b * g.kv_bs + (size_t)h * 64;
    const float* lse_b = lse + (size_t)bh * g.Nq;
    const float* delta_b = delta + (size_t)bh * g.Nq;

    const int k0 = tile_y * 128, kw = k0 + wave * 32, key = kw + col;
    const bool there = key < len;
    float* sums = sBias + blen * (1 + wave);
    for (int e = tid; e < 4 * blen; e += 256) sBias[blen + e] = 0.f;
    fill_bias(g, h, sBias, tid, 256);
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
    TileRegs<T> rq, rg;
    float rl = 0.f, rd = 0.f;
    auto prefetch = [&](int qt) {
        tile_load<T, true>(qb, (size_t)g.q_rs, qt, g.Nq, tid, rq);
        tile_load<T, true>(gb, (size_t)g.o_rs, qt, g.Nq, tid, rg);
        const int r = qt + (tid & 63) < g.Nq ? qt + (tid & 63) : g.Nq - 1;
        rl = lse_b[r];
        rd = delta_b[r];
    };
    if (q_lo < g.Nq) prefetch(q_lo);
    __syncthreads();
    const float far_past = sBias[0], far_ahead = sBias[blen - 1];
    for (int qt = q_lo; qt < g.Nq; qt += 64) {
        __syncthreads();
        tile_commit<T, true>(qt, g.Nq, tid, rq, sQ, sQt);
        tile_commit<T, true>(qt, g.Nq, tid, rg, sdO, sdOt);
        if (tid < 64) {
            const bool ok = qt + tid < g.Nq;
            sLse[tid] = ok ? rl : INFINITY;   // rows past the end weigh 0
            sDelta[tid] = ok ? rd : 0.f;
        }
        if (qt + 64 < g.Nq) prefetch(qt + 64);
        __syncthreads();
#pragma unroll
        for (int sb = 0; sb < 2; sb++) {
            const int first = start + qt + 32 * sb;   // position of the block's first query
            const bool past = kw + 31 - first <= -g.reach, ahead = kw - first - 31 >= g.reach;
            f16v s, dp = {};
            const int e0 = key - first - 4 * hi + span - 27;   // row r of the block: e0 + 27 - (r & 3) - 8 (r >> 2)
            if (past || ahead) {
                const float x = past ? far_past : far_ahead;
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = x;
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = sBias[e0 + (27 - (r & 3) - 8 * (r >> 2))];
            }
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                const vec8 aq = *reinterpret_cast<const vec8*>(&sQ[32 * sb + col][16 * ks + 8 * hi]);
                const vec8 ag = *reinterpret_cast<const vec8*>(&sdO[32 * sb + col][16 * ks + 8 * hi]);
                s = Tr<T>::mfma(aq, kf[ks], s);
                dp = Tr<T>::mfma(ag, vf[ks], dp);
            }
            if (kw + 32 > len || (g.causal && kw + 31 > first)) {
                const int least = !there ? 0x7fffffff : (g.causal ? key - first - 4 * hi : -64);   // the key's first row that sees it
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if ((r & 3) + 8 * (r >> 2) < least) s[r] = -INFINITY;
            }
            float ds[16];
            unsigned pp[8], pd[8];
#pragma unroll
            for (int g4 = 0; g4 < 4; g4++) {   // rows 8 g4 + 4 hi + {0 .. 3}
                const float4 L = *reinterpret_cast<const float4*>(&sLse[32 * sb + 8 * g4 + 4 * hi]);
                const float4 D = *reinterpret_cast<const float4*>(&sDelta[32 * sb + 8 * g4 + 4 * hi]);
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 0], g.c, -L.x)), p1 = __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 1], g.c, -L.y));
                const float p2 = __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 2], g.c, -L.z)), p3 = __builtin_amdgcn_exp2f(fmaf(s[4 * g4 + 3], g.c, -L.w));
                ds[4 * g4 + 0] = p0 * (dp[4 * g4 + 0] - D.x);
                ds[4 * g4 + 1] = p1 * (dp[4 * g4 + 1] - D.y);
                ds[4 * g4 + 2] = p2 * (dp[4 * g4 + 2] - D.z);
                ds[4 * g4 + 3] = p3 * (dp[4 * g4 + 3] - D.w);
                pp[2 * g4] = Tr<T>::pack2(p0, p1);
                pp[2 * g4 + 1] = Tr<T>::pack2(p2, p3);
                pd[2 * g4] = Tr<T>::pack2(ds[4 * g4], ds[4 * g4 + 1]);
                pd[2 * g4 + 1] = Tr<T>::pack2(ds[4 * g4 + 2], ds[4 * g4 + 3]);
            }
            if (past || ahead) {
                float x = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r++) x += ds[r];
                far_sum[past ? 0 : 1] += x;
            } else {
                // one half wave at a time: its 32 lanes are at 32 different distances; the other half's rows lie 4 further.  The array is this wave's own
                // and LDS operations of a wave keep their order, so the sums do too.
#pragma unroll
                for (int x = 0; x < 2; x++)
                    if (hi == x) {
#pragma unroll
                        for (int r = 0; r < 16; r++) __hip_atomic_fetch_add(&sums[e0 + (27 - (r & 3) - 8 * (r >> 2))], ds[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                    }
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; k2++) {
                const vec8 pf = packed_c_to_b_operand<T>(pp, k2), df = packed_c_to_b_operand<T>(pd, k2);
                const int qc = 32 * sb + 16 * k2 + 8 * hi;
                dv0 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sdOt[col][qc]), pf, dv0);
                dv1 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sdOt[32 + col][qc]), pf, dv1);
                dk0 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sQt[col][qc]), df, dk0);
                dk1 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sQt[32 + col][qc]), df, dk1);
            }
        }
    }
    if (key < g.Nk) {   // (behind the length: zeros)
        store_row<T>(dk + kvoff + (size_t)key * (size_t)g.kv_rs, dk0, dk1, g.scale, hi);
        store_row<T>(dv + kvoff + (size_t)key * (size_t)g.kv_rs, dv0, dv1, 1.0f, hi);
    }
    // distances into buckets
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float x = far_sum[i];
#pragma unroll
        for (int w = 32; w; w >>= 1) x += __shfl_xor(x, w, 64);
        if (lane == 0) sFar[wave][i] = x;
    }
    __syncthreads();
    for (int e = tid; e < blen; e += 256) sBias[e] = (sBias[blen + e] + sBias[2 * blen + e]) + (sBias[3 * blen + e] + sBias[4 * blen + e]);
    __syncthreads();
    if (tid < g.buckets) {
        const int k_ = tid < g.side ? tid : tid - g.side;   // bucket within its direction: distances lo .. hi of it
        const int lo = g.first[k_], up = k_ + 1 < g.side ? g.first[k_ + 1] - 1 : span;
        const float past = (sFar[0][0] + sFar[1][0]) + (sFar[2][0] + sFar[3][0]), ahead = (sFar[0][1] + sFar[1][1]) + (sFar[2][1] + sFar[3][1]);
        float x = 0.f;
        if (tid < g.side) {
            for (int n = lo; n <= up; n++) x += sBias[span - n];
            if (tid == g.side - 1) x += past;
            if (!g.both && tid == 0) {   // one direction: whatever lies ahead shares the bucket of distance 0
                for (int n = 1; n <= span; n++) x += sBias[span + n];
                x += ahead;
            }
        } else {
            for (int n = lo > 1 ? lo : 1; n <= up; n++) x += sBias[span + n];
            if (tid == g.buckets - 1) x += ahead;
        }
        part[((size_t)bh * gridDim.y + tile_y) * g.buckets + tid] = x;
    }
}

// Partial rows j = 0 .. count - 1 of head h lie at row ((j / tiles) H + h) tiles + j % tiles.  A wave a table entry, 64 bits, fixed order.
template <typename E>
__global__ void __launch_bounds__(64) k_rel_table(const float* __restrict__ part, E* __restrict__ dtable, int H, int buckets, int tiles, int count)
{
    const int bucket = blockIdx.x, h = blockIdx.y;
    double x = 0.0;
    for (int j = threadIdx.x; j < count; j += 64) x += (double)part[(((size_t)(j / tiles) * H + h) * tiles + j % tiles) * buckets + bucket];
#pragma unroll
    for (int w = 32; w; w >>= 1) x += __shfl_xor(x, w, 64);
    if (threadIdx.x == 0) dtable[bucket * H + h] = (E)(float)x;
}

// ---- up to 32 queries and keys -------------------------------------------------------------------------------------------------
// Both orientations of the score block are computed (a query per lane for dQ, delta and the table; a key per lane for dK and dV): 16 small products instead of a
// transposition through LDS; delta = sum_j P dP directly, O is not read.
template <typename T>
__global__ void __launch_bounds__(256, 2) k_rel_short_bwd(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ d_o,
                                                          const float* __restrict__ lse, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv,
                                                          float* __restrict__ part, int items, int waves)
{
    typedef typename Tr<T>::vec8 vec8;
    typedef T T2 __attribute__((ext_vector_type(2)));
    constexpr int TP = 40, OP = 72;
    __shared__ __attribute__((aligned(16))) T sQt[4][64][TP];
    __shared__ __attribute__((aligned(16))) T sKt[4][64][TP];
    __shared__ __attribute__((aligned(16))) T sGt[4][64][TP];
    __shared__ __attribute__((aligned(16))) T sO[4][32][OP];
    __shared__ __attribute__((aligned(16))) float sL[4][32];
    __shared__ __attribute__((aligned(16))) float sD[4][32];
    __shared__ float sB[4][64];
    __shared__ int sBk[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, r32 = lane & 31;
    const int gw = blockIdx.x * 4 + wave;
    if (gw >= waves) return;   // (no barriers below)
    const int h = gw % g.H, step = waves / g.H, nb = items / g.H, start = start_of(g, 0);
    const int qr = r32 < g.Nq ? r32 : g.Nq - 1;
    const int kp = lane & 15, vo = lane >> 4;
    const int q0r = 2 * kp < g.Nq ? 2 * kp : g.Nq - 1, q1r = 2 * kp + 1 < g.Nq ? 2 * kp + 1 : g.Nq - 1;
    sBk[wave][lane] = bucket_of(g, lane - 32 - start);
    sB[wave][lane] = start_value(g, table_at(g, sBk[wave][lane], h));   // distances -32 .. 31 less the start
    __builtin_amdgcn_wave_barrier();
    const float* bias_q = &sB[wave][4 * hi - r32 + 32];        // key row r: + (r & 3) + 8 (r >> 2)
    const float* bias_k = &sB[wave][r32 - 4 * hi + 32 - 27];   // query row r: + 27 - (r & 3) - 8 (r >> 2)
    f16v acc = {};   // dS^T summed over the wave's items

    vec8 qf[4], kf[4], vf[4], gf[4];
    auto load_ops = [&](int b) {
        const int n = len_of(g, b), last = n > 0 ? n - 1 : 0;
        const T* qb = q + (size_t)b * g.q_bs + (size_t)h * 64 + (size_t)qr * (size_t)g.q_rs + 8 * hi;
        const T* gb = d_o + (size_t)b * g.o_bs + (size_t)h * 64 + (size_t)qr * (size_t)g.o_rs + 8 * hi;
        const size_t kvb = (size_t)b * g.kv_bs + (size_t)h * 64 + (size_t)(r32 < last ? r32 : last) * (size_t)g.kv_rs + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            qf[ks] = *reinterpret_cast<const vec8*>(qb + 16 * ks);
            kf[ks] = *reinterpret_cast<const vec8*>(k + kvb + 16 * ks);
            vf[ks] = *reinterpret_cast<const vec8*>(v + kvb + 16 * ks);
            gf[ks] = *reinterpret_cast<const vec8*>(gb + 16 * ks);
        }
    };
    auto store_rows = [&](const f16v& x0, const f16v& x1, float mul, T* base, size_t rstride, int nrows) {
        store_row<T>(&sO[wave][r32][0], x0, x1, mul, hi);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int ps = 0; ps < 4; ps++) {
            const int row = (lane >> 3) + 8 * ps;
            const uint4 w = *reinterpret_cast<const uint4*>(&sO[wave][row][8 * (lane & 7)]);
            if (row < nrows) *reinterpret_cast<uint4*>(base + (size_t)row * rstride + 8 * (lane & 7)) = w;
        }
        __builtin_amdgcn_wave_barrier();
    };

    load_ops(gw / g.H);
    for (int b = gw / g.H; b < nb; b += step) {
        const int len = len_of(g, b), last = len > 0 ? len - 1 : 0;
        const size_t qbase = (size_t)b * g.q_bs + (size_t)h * 64, gbase = (size_t)b * g.o_bs + (size_t)h * 64, kbase = (size_t)b * g.kv_bs + (size_t)h * 64;
        const size_t k0r = (size_t)(2 * kp < last ? 2 * kp : last) * (size_t)g.kv_rs, k1r = (size_t)(2 * kp + 1 < last ? 2 * kp + 1 : last) * (size_t)g.kv_rs;
        vec8 xq[2][2], xk[2][2], xg[2][2];
#pragma unroll
        for (int ps = 0; ps < 2; ps++) {
            const int c = 8 * vo + 32 * ps;
            xk[ps][0] = *reinterpret_cast<const vec8*>(k + kbase + k0r + c);
            xk[ps][1] = *reinterpret_cast<const vec8*>(k + kbase + k1r + c);
            xq[ps][0] = *reinterpret_cast<const vec8*>(q + qbase + (size_t)q0r * (size_t)g.q_rs + c);
            xq[ps][1] = *reinterpret_cast<const vec8*>(q + qbase + (size_t)q1r * (size_t)g.q_rs + c);
            xg[ps][0] = *reinterpret_cast<const vec8*>(d_o + gbase + (size_t)q0r * (size_t)g.o_rs + c);
            xg[ps][1] = *reinterpret_cast<const vec8*>(d_o + gbase + (size_t)q1r * (size_t)g.o_rs + c);
        }
        const float L = r32 < g.Nq ? lse[((size_t)b * g.H + h) * g.Nq + qr] : INFINITY;   // (rows past the end weigh 0)
        if (len == 0) {   // row 0 was loaded, whatever it holds: a NaN times a weight of 0 would not be 0
#pragma unroll
            for (int ks = 0; ks < 4; ks++) { kf[ks] = vec8{}; vf[ks] = vec8{}; }
#pragma unroll
            for (int ps = 0; ps < 2; ps++) { xk[ps][0] = vec8{}; xk[ps][1] = vec8{}; }
        }
        // ---- a query per lane ----
        f16v sT, dpT = {};
#pragma unroll
        for (int r = 0; r < 16; r++) sT[r] = bias_q[(r & 3) + 8 * (r >> 2)];
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            sT = Tr<T>::mfma(kf[ks], qf[ks], sT);
            dpT = Tr<T>::mfma(vf[ks], gf[ks], dpT);
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
#pragma unroll
        for (int ps = 0; ps < 2; ps++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int ch = (vo + 4 * ps) * 8 + i;
                const T2 pk_ = { xk[ps][0][i], xk[ps][1][i] }, pq_ = { xq[ps][0][i], xq[ps][1][i] }, pg_ = { xg[ps][0][i], xg[ps][1][i] };
                *reinterpret_cast<T2*>(&sKt[wave][ch][2 * kp]) = pk_;
                *reinterpret_cast<T2*>(&sQt[wave][ch][2 * kp]) = pq_;
                *reinterpret_cast<T2*>(&sGt[wave][ch][2 * kp]) = pg_;
            }
        __builtin_amdgcn_wave_barrier();
        f16v a0 = {}, a1 = {};
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const vec8 df = packed_c_to_b_operand<T>(pdT, k2);
            a0 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sKt[wave][r32][16 * k2 + 8 * hi]), df, a0);
            a1 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sKt[wave][32 + r32][16 * k2 + 8 * hi]), df, a1);
        }
        // ---- a key per lane ----
        f16v s, dp = {};
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = bias_k[27 - (r & 3) - 8 * (r >> 2)];
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            s = Tr<T>::mfma(qf[ks], kf[ks], s);
            dp = Tr<T>::mfma(gf[ks], vf[ks], dp);
        }
        load_ops(b + step < nb ? b + step : b);   // in flight under everything below
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
            const vec8 pf = packed_c_to_b_operand<T>(pp, k2), df = packed_c_to_b_operand<T>(pd, k2);
            const int qc = 16 * k2 + 8 * hi;
            dv0 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sGt[wave][r32][qc]), pf, dv0);
            dv1 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sGt[wave][32 + r32][qc]), pf, dv1);
            dk0 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sQt[wave][r32][qc]), df, dk0);
            dk1 = Tr<T>::mfma(*reinterpret_cast<const vec8*>(&sQt[wave][32 + r32][qc]), df, dk1);
        }
        store_rows(dv0, dv1, 1.0f, dv + kbase, (size_t)g.kv_rs, g.Nk);
        store_rows(dk0, dk1, g.scale, dk + kbase, (size_t)g.kv_rs, g.Nk);
    }
    // dS^T by distance (a lane each: 31 at most on either side), then by bucket
    float* block = reinterpret_cast<float*>(&sO[wave][0][0]);   // [32 keys][33]
#pragma unroll
    for (int r = 0; r < 16; r++) block[((r & 3) + 8 * (r >> 2) + 4 * hi) * 33 + r32] = acc[r];
    __builtin_amdgcn_wave_barrier();
    float x = 0.f;
    for (int i = 0; i < 32; i++) {
        const int j = i + lane - 32;
        if (j >= 0 && j < 32) x += block[j * 33 + i];
    }
    sB[wave][lane] = x;
    __builtin_amdgcn_wave_barrier();
    for (int bucket = lane; bucket < g.buckets; bucket += 64) {
        float y = 0.f;
        for (int e = 0; e < 64; e++) y += sBk[wave][e] == bucket ? sB[wave][e] : 0.f;
        part[(size_t)gw * g.buckets + bucket] = y;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
bool is_short(const Geo& g) { return g.Nq <= 32 && g.Nk <= 32; }

// waves of the short form: what stays resident (LDS: one workgroup of 4 a CU), a multiple of the heads
int short_waves(const Geo& g, int B)
{
    long long waves = (long long)compute_units() * 4;
    if (waves > (long long)B * g.H) waves = (long long)B * g.H;
    return (int)(waves >= g.H ? waves / g.H * g.H : g.H);
}

long long partial_rows(const Geo& g, int B) { return is_short(g) ? short_waves(g, B) : (long long)B * g.H * ((g.Nk + 127) / 128); }

template <typename T>
int launch_bwd(const Geo& g, int B, const void* q, const void* k, const void* v, const void* out, const void* d_o, const float* lse, void* dq, void* dk, void* dv,
               void* dtable, float* ws, hipStream_t stream)
{
    const int BH = B * g.H;
    const long long rows = (long long)BH * g.Nq;
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
        if (BH > (1 << 23) || tiles > 65535 || qtiles > 65535 || (long long)B * tiles > 0x7fffffffLL) return fail(-1, "gvd_relattn_bwd: too many workgroups");
        count = B * tiles;
        const size_t lds = sizeof(float) * bias_len(g.reach);
        hipLaunchKernelGGL(k_rel_delta<T>, dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, stream, g, (const T*)out, (const T*)d_o, delta, rows);
        hipLaunchKernelGGL(k_rel_dq<T>, dim3((unsigned)BH, (unsigned)qtiles), dim3(256), lds, stream, g, (const T*)q, (const T*)k, (const T*)v, (const T*)d_o, lse, delta,
                           (T*)dq);
        hipLaunchKernelGGL(k_rel_dkv<T>, dim3((unsigned)BH, (unsigned)tiles), dim3(256), 5 * lds, stream, g, (const T*)q, (const T*)k, (const T*)v, (const T*)d_o, lse,
                           (const float*)delta, (T*)dk, (T*)dv, part);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(-2, "launch k_rel_*_bwd", e);
    const dim3 grid((unsigned)g.buckets, (unsigned)g.H);
#define GVD_TABLE(E) hipLaunchKernelGGL(k_rel_table<E>, grid, dim3(64), 0, stream, (const float*)part, (E*)dtable, g.H, g.buckets, tiles, count)
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
