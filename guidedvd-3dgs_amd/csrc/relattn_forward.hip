// relattn_forward.hip -- attention with a learned relative position bias, forward, for gfx950 (C-ABI: include/gvd_relattn.h).
//
//     s_ij = scale q_i . k_j + T[bucket(j - pos_i), h],  p = softmax over the keys seen,  o_i = sum_j p_ij v_j
//
// The bias is never laid out as [queries, keys]: buckets depend on the distance alone, so a workgroup expands its head's column of the table to one
// value a distance in LDS (a few hundred floats), and the products' ACCUMULATORS start from bias / scale instead of from zero: the scores leave
// the matrix unit with the bias in them.  A block of keys that lies entirely further than the last bucket's border starts from one constant.
//
//   k_rel_fwd     a wave = 32 or 64 queries, tiles of 64 keys through LDS, online softmax; optionally a part of the keys only (few rows: parts are
//                 joined by k_rel_join)
//   k_rel_short   up to 32 queries and keys (the frames of a pixel): a wave walks (batch, head) items, one pass over memory, no barriers
//   k_rel_few     up to 4 queries against many keys (new tokens against a cache): 8 lanes a key on the vector unit, bound by reading K and V once
#include <stdlib.h>

#include "relattn_common.h"

namespace gvdd {
thread_local std::string g_err;
int fail(int code, const char* what, hipError_t e)
{
    char buf[384];
    if (e != hipSuccess) snprintf(buf, sizeof buf, "%s: %s", what, hipGetErrorString(e));
    else snprintf(buf, sizeof buf, "%s", what);
    g_err = buf;
    return code;
}
}  // namespace gvdd

using namespace gvdr;

namespace gvdr {

int compute_units()
{
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    return cus;
}

int make_geo(const gvd_relattn_problem* p, Geo& g, const char* who)
{
    auto bad = [&](const char* what) {
        char buf[256];
        snprintf(buf, sizeof buf, "%s: %s", who, what);
        return fail(-1, buf);
    };
    if (!p) return bad("no problem given");
    if (p->B <= 0 || p->H <= 0 || p->Nq <= 0 || p->Nk <= 0) return bad("sizes must be positive");
    if ((long long)p->B * p->H > 0x7fffffffLL || p->Nq > (1 << 24) || p->Nk > (1 << 24)) return bad("too many (batch, head) items or rows");
    if ((long long)p->B * p->H * p->Nq > (1LL << 28)) return bad("too many rows of queries");
    if (p->D != 64) return bad("head dim must be 64");
    if (p->is_bf16 < 0 || p->is_bf16 > 1 || p->table_type < 0 || p->table_type > 2) return bad("unknown element type");
    if (p->buckets <= 0 || (p->both && p->buckets % 2)) return bad("buckets must be positive, and even where both directions have their own");
    const int side = p->both ? p->buckets / 2 : p->buckets;
    if (side > GVD_RELATTN_MAX_SIDE) return bad("too many buckets");
    if (!p->first || p->first[0] != 0) return bad("first[0] must be 0");
    for (int k = 1; k < side; k++)
        if (p->first[k] < p->first[k - 1]) return bad("first must not descend");
    if (p->first[side - 1] > GVD_RELATTN_MAX_REACH) return bad("the last bucket begins too far away");
    if (!(p->scale > 0.f) || !(p->scale < 1e30f) || !(p->scale > 1e-30f)) return bad("scale must be positive and within 1e-30 .. 1e30");
    if (p->q_start < -(1 << 29) || p->q_start > (1 << 29)) return bad("q_start is out of range");
    if ((p->q_bs | p->q_rs | p->kv_bs | p->kv_rs | p->o_bs | p->o_rs) & 7) return bad("strides must be multiples of 8 elements");
    g.H = p->H; g.Nq = p->Nq; g.Nk = p->Nk; g.buckets = p->buckets; g.side = side; g.both = p->both ? 1 : 0; g.causal = p->causal ? 1 : 0;
    g.reach = p->first[side - 1] > 1 ? p->first[side - 1] : 1;
    g.q_start = p->q_start; g.table_type = p->table_type;
    g.scale = p->scale; g.c = p->scale * LOG2E; g.inv_scale = 1.0f / p->scale;
    g.q_starts = p->q_starts; g.kv_lens = p->kv_lens; g.table = nullptr;
    g.q_bs = p->q_bs; g.q_rs = p->q_rs; g.kv_bs = p->kv_bs; g.kv_rs = p->kv_rs; g.o_bs = p->o_bs; g.o_rs = p->o_rs;
    for (int k = 0; k < GVD_RELATTN_MAX_SIDE; k++) g.first[k] = k < side ? p->first[k] : 0x7fffffff;
    return 0;
}

}  // namespace gvdr

namespace {

// What a row's weights are divided by, from their sum: 0 where the row sees nothing (its sum is 0 exactly, else at least one weight is about 1), and its log-sum-exp.
// A sum of NaN (a NaN or an infinity among the row's scores) stays one.
__device__ __forceinline__ float over(float sum) { return sum == 0.f ? 0.f : 1.0f / sum; }
__device__ __forceinline__ float lse_of(float max, float sum) { return sum == 0.f ? INFINITY : max + __builtin_amdgcn_logf(sum); }

// ---- general rows ------------------------------------------------------------------------------------------------------------
// Per query block and tile 32 exponentials a lane, with their products, roundings and sums some 770 cycles of a SIMD's vector unit, and 16 products of the matrix unit, 512 cycles.  The two take
// turns: at 9216 rows, 5 heads about 65 us of the one and 84 of the other (at a large product's rate), 134 to 145 us in all, 750 to 810 TFLOP/s; 20 heads 507, 860; 2304 rows, 10 heads: 31.7, with LSE 27 in a
// loop of training passes.  So the loop does little else:
//   * the maximum is not looked for: weights are formed with the running one, and a row sum above 2^15 (always for the first tile: the maximum starts
//     below every score) sends the block through the exact path.  Numerators and denominator share the maximum, so any one that keeps weights finite
//     gives the exact softmax;
//   * weights are rounded to the rows' type, the only operands that the matrix unit takes at this rate: half a step of each, 2^-11 or 2^-8, which the sum over keys averages (2.9e-4 of the
//     output's norm in fp16, 2.3e-3 in bf16; rounding the output alone leaves 2.1e-4 and 1.7e-3);
//   * each half wave keeps its own row sum, of the rounded weights (one dot product for two), or, where the backward will build on it (LSE), of the unrounded
//     ones: its weights sum to 1 in 32 bits then, which the table's gradient needs; the halves meet at the end;
//   * a block whose distances share one bias adds it to the exponent's shift, and its products start from the matrix unit's own zero.
//   * KS = 2: eight waves, two a SIMD where the grid gives a CU one workgroup only; the second four take every other tile of keys for the same rows and hand
//     maximum, sum and result over through LDS at the end.
template <typename T, int QB, bool PART, bool LSE, int KS>
__global__ void __launch_bounds__(256 * KS) __attribute__((amdgpu_waves_per_eu(2)))
k_rel_fwd(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ out, float* __restrict__ lse,
          float* __restrict__ part_o, float2* __restrict__ part_ml, int parts)
{
    typedef typename Tr<T>::vec8 vec8;
    constexpr int STAGE = KS * KV_TILE;   // keys between two barriers
    __shared__ __attribute__((aligned(16))) T sKb[2][STAGE][LDS_ROW];
    __shared__ __attribute__((aligned(16))) T sVb[2][STAGE][LDS_ROW];
    static_assert(KS == 1 || sizeof(sKb) + sizeof(sVb) >= 4 * QB * 34 * 64 * sizeof(float), "the hand-over uses the tiles' memory");
    extern __shared__ __attribute__((aligned(16))) float sBias[];

    int bh, tile_y;
    xcd_item_tile(bh, tile_y);
    const int qtile = PART ? tile_y / parts : tile_y, part = PART ? tile_y - qtile * parts : 0;
    const int b = bh / g.H, h = bh - b * g.H;
    const int tid = threadIdx.x, lane = tid & 63, wave8 = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wave8 & 3, hi = lane >> 5, col = lane & 31;
    const int k_off = KS == 1 ? 0 : KV_TILE * (wave8 >> 2);   // the wave's tile of a stage
    const int start = start_of(g, b), len = len_of(g, b);
    const T* qb = q + (size_t)b * g.q_bs + (size_t)h * 64;
    const T* kb = k + (size_t)b * g.kv_bs + (size_t)h * 64;
    const T* vb = v + (size_t)b * g.kv_bs + (size_t)h * 64;
    const int q0 = qtile * (128 * QB), q_last = (q0 + 128 * QB < g.Nq ? q0 + 128 * QB : g.Nq) - 1;
    // keys [k_lo, k_hi) are walked; those below k_full are seen by every row of the workgroup
    int k_lo = 0, k_hi = g.causal ? clamp_int(start + q_last + 1, 0, len) : len;
    const int k_full = g.causal ? clamp_int(start + q0 + 1, 0, len) : len;
    if (PART) {
        const int per = ((k_hi + STAGE - 1) / STAGE + parts - 1) / parts * STAGE;
        k_lo = part * per < k_hi ? part * per : k_hi;
        k_hi = k_lo + per < k_hi ? k_lo + per : k_hi;
    }

    int query[QB];
    vec8 qf[QB][4];
    f16v o0[QB], o1[QB];
    float m[QB], l[QB];   // l: of this half wave's keys
#pragma unroll
    for (int qi = 0; qi < QB; qi++) {
        query[qi] = q0 + (wave * QB + qi) * 32 + col;
        const T* qr = qb + (size_t)(query[qi] < g.Nq ? query[qi] : g.Nq - 1) * (size_t)g.q_rs + 8 * hi;   // (rows past the end: the last one again, not stored)
#pragma unroll
        for (int ks = 0; ks < 4; ks++) qf[qi][ks] = *reinterpret_cast<const vec8*>(qr + 16 * ks);
        o0[qi] = f16v{};
        o1[qi] = f16v{};
        m[qi] = LOWEST;
        l[qi] = 0.f;
    }

    // K and V tiles as they are, 16 bytes a lane, two passes; loads are issued a tile ahead.  Rows at or behind `len` are zeros (whatever lies there, also NaN,
    // meets a weight of 0): only the last tile looks.
    vec8 rk[2], rv[2];
    const int row = tid >> 3, c8 = (tid & 7) * 8;
    const size_t lane_off = (size_t)row * (size_t)g.kv_rs + c8, half_off = 32 * KS * (size_t)g.kv_rs;
    auto prefetch = [&](int kt) {
        const size_t base = (size_t)kt * (size_t)g.kv_rs;
        if (kt + STAGE <= len) {
#pragma unroll
            for (int ps = 0; ps < 2; ps++) {
                rk[ps] = *reinterpret_cast<const vec8*>(kb + base + (lane_off + ps * half_off));
                rv[ps] = *reinterpret_cast<const vec8*>(vb + base + (lane_off + ps * half_off));
            }
        } else {
#pragma unroll
            for (int ps = 0; ps < 2; ps++) {
                const int key = kt + row + 32 * KS * ps;
                const size_t off = (size_t)(key < len ? key : len - 1) * (size_t)g.kv_rs + c8;
                rk[ps] = *reinterpret_cast<const vec8*>(kb + off);
                rv[ps] = *reinterpret_cast<const vec8*>(vb + off);
                if (key >= len) { rk[ps] = vec8{}; rv[ps] = vec8{}; }
            }
        }
    };
    auto commit = [&](int buf) {
#pragma unroll
        for (int ps = 0; ps < 2; ps++) {
            *reinterpret_cast<vec8*>(&sKb[buf][row + 32 * KS * ps][c8]) = rk[ps];
            *reinterpret_cast<vec8*>(&sVb[buf][row + 32 * KS * ps][c8]) = rv[ps];
        }
    };
    if (k_lo < k_hi) prefetch(k_lo);
    fill_bias(g, h, sBias, tid, 256 * KS);
    float far_past = 0.f, far_ahead = 0.f;

    auto tile = [&](int stage, int buf, auto masked_tag) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        if (stage + STAGE < k_hi) {
            commit(buf ^ 1);
            if (stage + 2 * STAGE < k_hi) prefetch(stage + 2 * STAGE);
        }
        const int kt = stage + k_off;
        const T (*sK)[LDS_ROW] = sKb[buf] + k_off;
        f16v s0[QB], s1[QB];
        float far[QB];   // the single bias of a far block, in the exponent
        vec8 a0[4], a1[4];
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            a0[ks] = *reinterpret_cast<const vec8*>(&sK[col][16 * ks + 8 * hi]);
            a1[ks] = *reinterpret_cast<const vec8*>(&sK[32 + col][16 * ks + 8 * hi]);
        }
#pragma unroll
        for (int qi = 0; qi < QB; qi++) {
            const int first = start + q0 + (wave * QB + qi) * 32;   // position of the block's first query (uniform)
            if (kt + 63 - first <= -g.reach || kt - first - 31 >= g.reach) {
                far[qi] = kt < first ? far_past : far_ahead;
                s0[qi] = Tr<T>::mfma(a0[0], qf[qi][0], f16v{});
                s1[qi] = Tr<T>::mfma(a1[0], qf[qi][0], f16v{});
            } else {
                far[qi] = 0.f;
                const float* e = sBias + (kt + 4 * hi - first - col + g.reach + PAD);
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s0[qi][r] = e[(r & 3) + 8 * (r >> 2)];
                    s1[qi][r] = e[(r & 3) + 8 * (r >> 2) + 32];
                }
                s0[qi] = Tr<T>::mfma(a0[0], qf[qi][0], s0[qi]);
                s1[qi] = Tr<T>::mfma(a1[0], qf[qi][0], s1[qi]);
            }
        }
#pragma unroll
        for (int ks = 1; ks < 4; ks++)
#pragma unroll
            for (int qi = 0; qi < QB; qi++) {
                s0[qi] = Tr<T>::mfma(a0[ks], qf[qi][ks], s0[qi]);
                s1[qi] = Tr<T>::mfma(a1[ks], qf[qi][ks], s1[qi]);
            }
        unsigned pk0[QB][8], pk1[QB][8];
#pragma unroll
        for (int qi = 0; qi < QB; qi++) {
            if (MASKED) {
                const int seen = (g.causal && start + query[qi] + 1 < len ? start + query[qi] + 1 : len) - kt - 4 * hi;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    if ((r & 3) + 8 * (r >> 2) >= seen) s0[qi][r] = -INFINITY;
                    if ((r & 3) + 8 * (r >> 2) + 32 >= seen) s1[qi][r] = -INFINITY;
                }
            }
            auto weights = [&]() {   // and this half's sum of them
                const float shift = far[qi] - m[qi];
                float x = 0.f, y = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s0[qi][2 * j], g.c, shift)), p1 = __builtin_amdgcn_exp2f(fmaf(s0[qi][2 * j + 1], g.c, shift));
                    const float p2 = __builtin_amdgcn_exp2f(fmaf(s1[qi][2 * j], g.c, shift)), p3 = __builtin_amdgcn_exp2f(fmaf(s1[qi][2 * j + 1], g.c, shift));
                    pk0[qi][j] = Tr<T>::pack2(p0, p1);
                    pk1[qi][j] = Tr<T>::pack2(p2, p3);
                    x = LSE ? x + (p0 + p1) : add_pair<T>(pk0[qi][j], x);
                    y = LSE ? y + (p2 + p3) : add_pair<T>(pk1[qi][j], y);
                }
                return x + y;
            };
            float sum = weights();
            if (__any(!(sum <= 32768.f))) {   // (an infinity or a NaN too)
                float mt = fmaxf(s0[qi][0], s1[qi][0]);
#pragma unroll
                for (int r = 1; r < 16; r++) mt = max3f(mt, s0[qi][r], s1[qi][r]);
                mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
                const float m_new = fmaxf(m[qi], fmaf(mt, g.c, far[qi])), alpha = __builtin_amdgcn_exp2f(m[qi] - m_new);
                m[qi] = m_new;
                l[qi] *= alpha;
#pragma unroll
                for (int r = 0; r < 16; r++) { o0[qi][r] *= alpha; o1[qi][r] *= alpha; }
                sum = weights();
            }
            l[qi] += sum;
        }
#pragma unroll
        for (int kbk = 0; kbk < 2; kbk++)
#pragma unroll
            for (int k2 = 0; k2 < 2; k2++) {
                const vec8 v0 = transposed_operand(&sVb[buf][0][0], LDS_ROW, k_off + 32 * kbk + 16 * k2, 0, lane);
                const vec8 v1 = transposed_operand(&sVb[buf][0][0], LDS_ROW, k_off + 32 * kbk + 16 * k2, 32, lane);
#pragma unroll
                for (int qi = 0; qi < QB; qi++) {
                    const vec8 pf = packed_operand<T>(kbk == 0 ? pk0[qi] : pk1[qi], k2);
                    o0[qi] = Tr<T>::mfma(v0, pf, o0[qi]);
                    o1[qi] = Tr<T>::mfma(v1, pf, o1[qi]);
                }
            }
        __syncthreads();
    };

    if (k_lo < k_hi) {   // (uniform over the workgroup)
        commit(0);
        if (k_lo + STAGE < k_hi) prefetch(k_lo + STAGE);
        __syncthreads();
        far_past = sBias[0] * g.c;
        far_ahead = sBias[bias_len(g.reach) - 1] * g.c;
        int kt = k_lo, buf = 0;
        for (; kt < k_hi && kt + STAGE <= k_full; kt += STAGE, buf ^= 1) tile(kt, buf, std::false_type{});
        for (; kt < k_hi; kt += STAGE, buf ^= 1) tile(kt, buf, std::true_type{});
    }
#pragma unroll
    for (int qi = 0; qi < QB; qi++) l[qi] += __shfl_xor(l[qi], 32, 64);
    if (KS == 2) {   // (the loop's last barrier lies behind all reads of the tiles)
        auto at = [&](int qi) { float* base = reinterpret_cast<float*>(qi % 2 ? &sVb[0][0][0] : &sKb[0][0][0]); return base + (wave * 34) * 64 + lane; };
        if (wave8 >= 4) {
#pragma unroll
            for (int qi = 0; qi < QB; qi++) {
                float* x = at(qi);
#pragma unroll
                for (int r = 0; r < 16; r++) { x[64 * r] = o0[qi][r]; x[64 * (16 + r)] = o1[qi][r]; }
                x[64 * 32] = m[qi];
                x[64 * 33] = l[qi];
            }
        }
        __syncthreads();
        if (wave8 >= 4) return;
#pragma unroll
        for (int qi = 0; qi < QB; qi++) {
            const float* x = at(qi);
            const float m1 = x[64 * 32], top = fmaxf(m[qi], m1), w0 = __builtin_amdgcn_exp2f(m[qi] - top), w1 = __builtin_amdgcn_exp2f(m1 - top);
            m[qi] = top;
            l[qi] = l[qi] * w0 + x[64 * 33] * w1;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                o0[qi][r] = o0[qi][r] * w0 + x[64 * r] * w1;
                o1[qi][r] = o1[qi][r] * w0 + x[64 * (16 + r)] * w1;
            }
        }
    }
#pragma unroll
    for (int qi = 0; qi < QB; qi++) {
        if (query[qi] >= g.Nq) continue;
        if (PART) {
            const size_t row = ((size_t)part * (gridDim.x) + bh) * g.Nq + query[qi];
            if (hi == 0) part_ml[row] = make_float2(m[qi], l[qi]);
            float* po = part_o + row * 64;
#pragma unroll
            for (int rg = 0; rg < 4; rg++) {
                const int d0 = 8 * rg + 4 * hi;
                *reinterpret_cast<float4*>(po + d0) = make_float4(o0[qi][4 * rg], o0[qi][4 * rg + 1], o0[qi][4 * rg + 2], o0[qi][4 * rg + 3]);
                *reinterpret_cast<float4*>(po + 32 + d0) = make_float4(o1[qi][4 * rg], o1[qi][4 * rg + 1], o1[qi][4 * rg + 2], o1[qi][4 * rg + 3]);
            }
            continue;
        }
        if (LSE && hi == 0) lse[(size_t)bh * g.Nq + query[qi]] = lse_of(m[qi], l[qi]);
        const float inv = over(l[qi]);
        T* orow = out + (size_t)b * g.o_bs + (size_t)h * 64 + (size_t)query[qi] * (size_t)g.o_rs;
#pragma unroll
        for (int rg = 0; rg < 4; rg++) {
            const int d0 = 8 * rg + 4 * hi;
            uint2 w0, w1;
            w0.x = Tr<T>::pack2(o0[qi][4 * rg] * inv, o0[qi][4 * rg + 1] * inv);
            w0.y = Tr<T>::pack2(o0[qi][4 * rg + 2] * inv, o0[qi][4 * rg + 3] * inv);
            w1.x = Tr<T>::pack2(o1[qi][4 * rg] * inv, o1[qi][4 * rg + 1] * inv);
            w1.y = Tr<T>::pack2(o1[qi][4 * rg + 2] * inv, o1[qi][4 * rg + 3] * inv);
            *reinterpret_cast<uint2*>(orow + d0) = w0;
            *reinterpret_cast<uint2*>(orow + 32 + d0) = w1;
        }
    }
}

// Joins the parts of a row: LN lanes a row, its 64 channels on 16 of them, LN / 16 parts at once.  64 lanes where rows are few (the trips to memory count: 16 x 10
// rows in 13 parts 4.5 us, with 16 lanes 8.9), 16 where they are many (46080 rows in 3 parts 9.4 us, with 64 lanes 16.9).
template <typename T, int LN>
__global__ void __launch_bounds__(256) k_rel_join(const Geo g, const float* __restrict__ part_o, const float2* __restrict__ part_ml, int parts, int BH,
                                                  T* __restrict__ out, float* __restrict__ lse)
{
    constexpr int CH = 64 / LN;   // parts come in CH rounds of LN: lane s of a round holds part s's maximum and sum (up to 64 parts)
    const long long row = (long long)blockIdx.x * (256 / LN) + threadIdx.x / LN, rows = (long long)BH * g.Nq;
    if (row >= rows) return;
    const int lane = threadIdx.x % LN, d0 = (lane & 15) * 4;
    float2 ml[CH];
    float top = LOWEST, total = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int s = c * LN + lane;
        ml[c] = s < parts ? part_ml[(size_t)s * rows + row] : make_float2(LOWEST, 0.f);
        top = fmaxf(top, ml[c].x);
    }
#pragma unroll
    for (int w = LN / 2; w; w >>= 1) top = fmaxf(top, __shfl_xor(top, w, LN));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < CH; c++) {
        if (c * LN >= parts) break;
        const float weight = __builtin_amdgcn_exp2f(ml[c].x - top);
        total = fmaf(weight, ml[c].y, total);
        const int n = parts - c * LN < LN ? parts - c * LN : LN;
        for (int s0 = 0; s0 < n; s0 += LN / 16) {
            const int s = s0 + (lane >> 4);
            const float w = __shfl(weight, s, LN);
            if (s < n) {
                const float4 x = *reinterpret_cast<const float4*>(part_o + ((size_t)(c * LN + s) * rows + row) * 64 + d0);
                o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
            }
        }
    }
#pragma unroll
    for (int w = LN / 2; w; w >>= 1) total += __shfl_xor(total, w, LN);
#pragma unroll
    for (int w = 16; w < LN; w <<= 1) {
        o.x += __shfl_xor(o.x, w, LN); o.y += __shfl_xor(o.y, w, LN);
        o.z += __shfl_xor(o.z, w, LN); o.w += __shfl_xor(o.w, w, LN);
    }
    const float inv = over(total);
    if (lane < 16) {
        const long long bh = row / g.Nq;
        const int n = (int)(row - bh * g.Nq), b = (int)(bh / g.H), h = (int)(bh - (long long)b * g.H);
        uint2 w;
        w.x = Tr<T>::pack2(o.x * inv, o.y * inv);
        w.y = Tr<T>::pack2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(out + (size_t)b * g.o_bs + (size_t)n * g.o_rs + (size_t)h * 64 + d0) = w;
        if (lse && lane == 0) lse[row] = lse_of(top, total);
    }
}

// ---- up to 32 queries and keys -------------------------------------------------------------------------------------------------
// The whole problem of an item is 3 x 32 x 128 bytes in and 32 x 128 out: memory.  A wave keeps one head (its stride over items is a multiple of H),
// so its 16 biases a lane stay in registers over all its items (from 33 queries or keys on there is no such form); the next item's rows are requested as soon as this one's registers are free.  Rows are
// read whole, 8 lanes each, and take their operand forms through one piece of LDS, Q then K then V then the result (LDS operations of a wave keep their order).
template <typename T>
__global__ void __launch_bounds__(256) k_rel_short(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ out,
                                                   float* __restrict__ lse, int items, int waves)
{
    typedef typename Tr<T>::vec8 vec8;
    constexpr int PITCH = 72;
    __shared__ __attribute__((aligned(16))) T sRows[4][32][PITCH];
    __shared__ float sB[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, r32 = lane & 31;
    const int gw = blockIdx.x * 4 + wave;
    if (gw >= waves) return;   // (no barriers below)
    const int h = gw % g.H, step = waves / g.H, nb = items / g.H;
    const int row = lane >> 3, c8 = 8 * (lane & 7);   // rows 8 i + row
    T (*rows)[PITCH] = sRows[wave];
    vec8 rq[4], rk[4], rv[4];
    int len_next;
    // rows at or behind the length: the last one again; their scores are masked.  (A length of zero: row 0, and the item's result is zeros.)
    auto load = [&](int b) {
        len_next = len_of(g, b);
        const int last = len_next > 0 ? len_next - 1 : 0;
        const T* qb = q + (size_t)b * g.q_bs + (size_t)h * 64 + c8;
        const size_t kv = (size_t)b * g.kv_bs + (size_t)h * 64 + c8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + row;
            rq[i] = *reinterpret_cast<const vec8*>(qb + (size_t)(r < g.Nq ? r : g.Nq - 1) * (size_t)g.q_rs);
            const size_t off = kv + (size_t)(r < last ? r : last) * (size_t)g.kv_rs;
            rk[i] = *reinterpret_cast<const vec8*>(k + off);
            rv[i] = *reinterpret_cast<const vec8*>(v + off);
        }
    };
    auto put = [&](const vec8 (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<vec8*>(&rows[8 * i + row][c8]) = x[i];
        wave_order();
    };
    f16v bias;
    int biased = 0x7fffffff;   // the start that `bias` is for
    auto set_bias = [&](int start) {
        sB[wave][lane] = start_value(g, table_at(g, bucket_of(g, lane - 32 - start), h));   // distances -32 .. 31 less the start
        wave_order();
#pragma unroll
        for (int r = 0; r < 16; r++) bias[r] = sB[wave][(r & 3) + 8 * (r >> 2) + 4 * hi - r32 + 32];
        wave_order();
        biased = start;
    };
    load(gw / g.H);
    for (int b = gw / g.H; b < nb; b += step) {
        const int len = len_next, start = start_of(g, b);
        if (start != biased) set_bias(start);
        vec8 qf[4], kf[4];
        put(rq);
#pragma unroll
        for (int ks = 0; ks < 4; ks++) qf[ks] = *reinterpret_cast<const vec8*>(&rows[r32][16 * ks + 8 * hi]);
        wave_order();
        put(rk);
#pragma unroll
        for (int ks = 0; ks < 4; ks++) kf[ks] = *reinterpret_cast<const vec8*>(&rows[r32][16 * ks + 8 * hi]);
        wave_order();
        put(rv);
        load(b + step < nb ? b + step : b);
        f16v s = bias;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) s = Tr<T>::mfma(kf[ks], qf[ks], s);
        const int seen = (g.causal && start + r32 + 1 < len ? start + r32 + 1 : len) - 4 * hi;
#pragma unroll
        for (int r = 0; r < 16; r++)
            if ((r & 3) + 8 * (r >> 2) >= seen) s[r] = -INFINITY;
        float mt = max3f(s[0], s[1], s[2]);
#pragma unroll
        for (int r = 3; r < 15; r += 2) mt = max3f(mt, s[r], s[r + 1]);
        mt = fmaxf(mt, s[15]);
        mt = fmaxf(fmaxf(mt, __shfl_xor(mt, 32, 64)) * g.c, LOWEST);
        unsigned pk[8];
        float l = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * j], g.c, -mt)), p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * j + 1], g.c, -mt));
            pk[j] = Tr<T>::pack2(p0, p1);
            l += p0 + p1;
        }
        l += __shfl_xor(l, 32, 64);
        f16v o0 = {}, o1 = {};
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const vec8 pf = packed_operand<T>(pk, k2);
            o0 = Tr<T>::mfma(transposed_operand(&rows[0][0], PITCH, 16 * k2, 0, lane), pf, o0);
            o1 = Tr<T>::mfma(transposed_operand(&rows[0][0], PITCH, 16 * k2, 32, lane), pf, o1);
        }
        wave_order();
        const bool empty = l == 0.f;   // (its result is not formed as 0 times what was summed: with a length of zero row 0 of V was loaded, whatever it holds)
        if (lse && hi == 0 && r32 < g.Nq) lse[((size_t)b * g.H + h) * g.Nq + r32] = lse_of(mt, l);
        const float inv = 1.0f / l;
#pragma unroll
        for (int rg = 0; rg < 4; rg++) {
            const int d0 = 8 * rg + 4 * hi;
            uint2 w0, w1;
            w0.x = Tr<T>::pack2(o0[4 * rg] * inv, o0[4 * rg + 1] * inv);
            w0.y = Tr<T>::pack2(o0[4 * rg + 2] * inv, o0[4 * rg + 3] * inv);
            w1.x = Tr<T>::pack2(o1[4 * rg] * inv, o1[4 * rg + 1] * inv);
            w1.y = Tr<T>::pack2(o1[4 * rg + 2] * inv, o1[4 * rg + 3] * inv);
            if (empty) { w0 = make_uint2(0, 0); w1 = make_uint2(0, 0); }
            *reinterpret_cast<uint2*>(&rows[r32][d0]) = w0;
            *reinterpret_cast<uint2*>(&rows[r32][32 + d0]) = w1;
        }
        wave_order();
        T* ob = out + (size_t)b * g.o_bs + (size_t)h * 64 + c8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + row;
            const u4 w = *reinterpret_cast<const u4*>(&rows[r][c8]);
            if (r < g.Nq) __builtin_nontemporal_store(w, reinterpret_cast<u4*>(ob + (size_t)r * (size_t)g.o_rs));
        }
        wave_order();
    }
}

// ---- few queries, many keys ----------------------------------------------------------------------------------------------------
// 8 lanes hold a key's 64 channels, a wave 8 keys at once, 4 of those in flight; every lane group keeps its own running maximum and sum, joined at the end.
// 16 x 10 rows against caches of 8192 (half full on average): 37 us with the join, 4.8 TB/s.  (When these were tried it was 41: with ordinary loads 45, with an item's
// parts on one XCD 3 more, with 8 workgroups a CU 41 -- and 64 x 20 rows against 1000: 39 against 36 --, with 8 keys a lane group in flight 63.)
template <typename T, int NQ>
__global__ void __launch_bounds__(256) k_rel_few(const Geo g, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ out,
                                                 float* __restrict__ lse, float* __restrict__ part_o, float2* __restrict__ part_ml, int parts)
{
    typedef typename Tr<T>::vec8 vec8;
    constexpr int U = 4;
    __shared__ float sO[4][NQ][64];
    __shared__ float sM[4][NQ], sL[4][NQ];
    extern __shared__ __attribute__((aligned(16))) float sBias[];
    const int bh = blockIdx.x, part = blockIdx.y;   // the heads of a key lie next to each other: their workgroups run at once
    const int b = bh / g.H, h = bh - b * g.H;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = lane >> 3, sub = lane & 7;
    const int start = start_of(g, b), len = len_of(g, b);
    const int k_end = g.causal ? clamp_int(start + g.Nq, 0, len) : len;
    const int per = ((k_end + 127) / 128 + parts - 1) / parts * 128;
    const int k_lo = part * per < k_end ? part * per : k_end, k_hi = k_lo + per < k_end ? k_lo + per : k_end;
    const T* kb = k + (size_t)b * g.kv_bs + (size_t)h * 64 + 8 * sub;
    const T* vb = v + (size_t)b * g.kv_bs + (size_t)h * 64 + 8 * sub;
    vec8 kf[U], vf[U];
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = base + 8 * u + grp;
            const size_t off = (size_t)(j < k_hi ? j : k_hi - 1) * (size_t)g.kv_rs;
            kf[u] = __builtin_nontemporal_load(reinterpret_cast<const vec8*>(kb + off));
            vf[u] = __builtin_nontemporal_load(reinterpret_cast<const vec8*>(vb + off));
        }
    };
    const int base0 = k_lo + wave * 32;
    if (base0 < k_hi) load(base0);
    float qv[NQ][8], acc[NQ][8], m[NQ], l[NQ];
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const vec8 x = *reinterpret_cast<const vec8*>(q + (size_t)b * g.q_bs + (size_t)(i < g.Nq ? i : g.Nq - 1) * (size_t)g.q_rs + (size_t)h * 64 + 8 * sub);
#pragma unroll
        for (int e = 0; e < 8; e++) { qv[i][e] = (float)x[e]; acc[i][e] = 0.f; }
        m[i] = LOWEST;
        l[i] = 0.f;
    }
    fill_bias(g, h, sBias, tid, 256);
    __syncthreads();
    const int span = g.reach + PAD;
    for (int base = base0; base < k_hi; base += 128) {
        float kk[U][8], vv[U][8];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) { kk[u][e] = (float)kf[u][e]; vv[u][e] = (float)vf[u][e]; }
        if (base + 128 < k_hi) load(base + 128);
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            float s[U], top = m[i];
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) x = fmaf(qv[i][e], kk[u][e], x);
                x += __shfl_xor(x, 1, 64);
                x += __shfl_xor(x, 2, 64);
                x += __shfl_xor(x, 4, 64);
                const int j = base + 8 * u + grp, d = j - start - i;
                x = (x + sBias[clamp_int(d, -span, span) + span]) * g.c;
                s[u] = j < k_hi && !(g.causal && d > 0) ? x : -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float alpha = __builtin_amdgcn_exp2f(m[i] - top);
            m[i] = top;
            l[i] *= alpha;
            float p[U];
#pragma unroll
            for (int u = 0; u < U; u++) { p[u] = __builtin_amdgcn_exp2f(s[u] - top); l[i] += p[u]; }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float a = acc[i][e] * alpha;
#pragma unroll
                for (int u = 0; u < U; u++) a = fmaf(p[u], vv[u][e], a);
                acc[i][e] = a;
            }
        }
    }
    // join the wave's 8 lane groups, then the workgroup's 4 waves
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        float top = m[i];
#pragma unroll
        for (int x = 8; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        const float w = __builtin_amdgcn_exp2f(m[i] - top);
        float sum = l[i] * w;
#pragma unroll
        for (int x = 8; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float a = acc[i][e] * w;
#pragma unroll
            for (int x = 8; x < 64; x <<= 1) a += __shfl_xor(a, x, 64);
            if (grp == 0) sO[wave][i][8 * sub + e] = a;
        }
        if (lane == 0) { sM[wave][i] = top; sL[wave][i] = sum; }
    }
    __syncthreads();
    for (int t = tid; t < NQ * 64; t += 256) {
        const int i = t >> 6, d = t & 63;
        if (i >= g.Nq) continue;
        const float top = fmaxf(fmaxf(sM[0][i], sM[1][i]), fmaxf(sM[2][i], sM[3][i]));
        float total = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(sM[w][i] - top);
            total = fmaf(f, sL[w][i], total);
            o = fmaf(f, sO[w][i][d], o);
        }
        if (parts > 1) {
            const size_t row = ((size_t)part * gridDim.x + bh) * g.Nq + i;
            part_o[row * 64 + d] = o;
            if (d == 0) part_ml[row] = make_float2(top, total);
        } else {
            out[(size_t)b * g.o_bs + (size_t)i * g.o_rs + (size_t)h * 64 + d] = (T)(total == 0.f ? 0.f : o / total);
            if (lse && d == 0) lse[(size_t)bh * g.Nq + i] = lse_of(top, total);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
enum Form { SHORT, FEW, GENERAL };

struct Plan { Form form; int qb, tiles, parts, ks; };

// Which kernel, how many query blocks a wave, and into how many parts the keys are cut.
// General rows: what a choice takes is estimated, in microseconds, and the least is taken.  A workgroup of 128 rows takes 0.95 a tile alone on its CU and 0.745 with
// others, one of 256 rows 1.5 and 1.3 (their K and V fragments serve twice the products), one of 128 rows and eight waves 1.48 for two tiles, alone (with others there it has
// nothing to gain: 2304, 20 heads 61.5 against 58); a round of workgroups starts with 4 (bias, first tiles), with eight waves 5; parts
// take 8 (their stores, the join's launch) and 3.3e-5 a row and part.  Measured, with the join (us): 9216 queries and keys, 5 heads: 128 rows 212, in 2 parts 162; 256 rows 212, in 2 parts
// 186, in 4 parts 157.  2304, 10 heads: 128 rows 37, with eight waves 31.7, 256 rows 55, 128 rows in 2 parts 42.  1024, 80 items: 128 rows 41, in 2 parts 53; 256 rows 48.  Over ten
// shapes and eight choices each, what it picks is 0.5 % off the best on average, 3 % at most.
Plan plan_of(const Geo& g, int B, int cus)
{
    const long long bh = (long long)B * g.H;
    if (g.Nq <= 32 && g.Nk <= 32) return { SHORT, 1, 1, 1, 1 };
    if (g.Nq <= 4) {   // few rows: 4 workgroups a CU, at least 256 keys each
        long long parts = ((long long)cus * 4 + bh - 1) / bh;
        const long long most = (g.Nk + 255) / 256;
        if (parts > most) parts = most;
        return { FEW, 1, 1, (int)(parts < 64 ? parts : 64), 1 };
    }
    Plan best = { GENERAL, 1, 1, 1, 1 };
    double least = 1e30;
    const int tiles = (g.Nk + KV_TILE - 1) / KV_TILE;
    for (int qb = 1; qb <= 2; qb++) {
        const int rows = 128 * qb, qtiles = (g.Nq + rows - 1) / rows;
        for (int parts = 1; parts <= 64 && (parts == 1 || 2 * parts <= tiles); parts++) {
            const double load = (double)bh * qtiles * parts / cus, rounds = load <= 1.0 ? 1.0 : (load < 8.0 ? __builtin_ceil(load) : load);
            const double a_tile = rounds == 1.0 ? (qb == 2 ? 1.5 : 0.95) : rounds * (qb == 2 ? 1.3 : 0.745);
            const double t = 4.0 * rounds + (tiles + parts - 1) / parts * a_tile + (parts > 1 ? 8.0 + 3.3e-5 * (double)bh * g.Nq * parts : 0.0);
            if (t < least) { least = t; best = { GENERAL, qb, qtiles, parts, 1 }; }
            if (qb == 2 || rounds > 1.0) continue;
            const int stages = (tiles + 1) / 2;   // of 128 keys
            const double t2 = 5.0 + (stages + parts - 1) / parts * 1.48 + (t - 4.0 * rounds - (tiles + parts - 1) / parts * a_tile);
            if (t2 < least) { least = t2; best = { GENERAL, 1, qtiles, parts, 2 }; }
        }
    }
    return best;
}

size_t part_rows(const Geo& g, int B, const Plan& pl) { return (size_t)pl.parts * B * g.H * g.Nq; }

template <typename T>
int launch_fwd(const Geo& g, int B, const void* q, const void* k, const void* v, void* out, float* lse, void* ws, hipStream_t stream)
{
    const int cus = compute_units();
    const Plan pl = plan_of(g, B, cus);
    const int BH = B * g.H;
    if (pl.form != SHORT && (BH > (1 << 23) || (long long)pl.tiles * pl.parts > 65535 || (long long)BH * pl.tiles * pl.parts > 0x7fffffffLL))
        return fail(-1, "gvd_relattn_fwd: too many workgroups");
    float* po = nullptr;
    float2* ml = nullptr;
    if (pl.parts > 1) {
        if (!ws) return fail(-1, "gvd_relattn_fwd: this problem needs a workspace");
        if ((uintptr_t)ws & 15) return fail(-1, "gvd_relattn_fwd: the workspace must be 16-byte aligned");
        po = (float*)ws;
        ml = (float2*)(po + part_rows(g, B, pl) * 64);
    }
    const size_t lds = sizeof(float) * bias_len(g.reach);
    if (pl.form == SHORT) {
        // 8 waves a CU, a multiple of the heads (46080 items of 25 frames: 118.7 us; with 4 115.8, 12 127, 16 123; 11200 items with the backward: 101, 4 110, 16 102)
        long long waves = (long long)cus * 8;
        if (waves > BH) waves = BH;
        waves = waves >= g.H ? waves / g.H * g.H : g.H;
        hipLaunchKernelGGL(k_rel_short<T>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream, g, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, BH, (int)waves);
    } else if (pl.form == FEW) {
        const dim3 grid((unsigned)BH, (unsigned)pl.parts);
#define GVD_FEW(N) hipLaunchKernelGGL((k_rel_few<T, N>), grid, dim3(256), lds, stream, g, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, po, ml, pl.parts)
        if (g.Nq == 1) GVD_FEW(1); else if (g.Nq == 2) GVD_FEW(2); else GVD_FEW(4);
#undef GVD_FEW
    } else {
        const dim3 grid((unsigned)BH, (unsigned)(pl.tiles * pl.parts));
#define GVD_GEN(Q, P, K) if (lse) GVD_GEN_(Q, P, true, K); else GVD_GEN_(Q, P, false, K)
#define GVD_GEN_(Q, P, L, K) hipLaunchKernelGGL((k_rel_fwd<T, Q, P, L, K>), grid, dim3(256 * K), lds, stream, g, (const T*)q, (const T*)k, (const T*)v, (T*)out, lse, po, ml, pl.parts)
        if (pl.ks == 2 && pl.parts > 1) { GVD_GEN(1, true, 2); }
        else if (pl.ks == 2) { GVD_GEN(1, false, 2); }
        else if (pl.qb == 2 && pl.parts > 1) { GVD_GEN(2, true, 1); }
        else if (pl.qb == 2) { GVD_GEN(2, false, 1); }
        else if (pl.parts > 1) { GVD_GEN(1, true, 1); }
        else { GVD_GEN(1, false, 1); }
#undef GVD_GEN
#undef GVD_GEN_
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(-2, "launch k_rel_*", e);
    if (pl.parts > 1) {
        const long long rows = (long long)BH * g.Nq;
        if (rows < 4096)
            hipLaunchKernelGGL((k_rel_join<T, 64>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, g, po, ml, pl.parts, BH, (T*)out, lse);
        else
            hipLaunchKernelGGL((k_rel_join<T, 16>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, stream, g, po, ml, pl.parts, BH, (T*)out, lse);
        e = hipGetLastError();
        if (e != hipSuccess) return fail(-2, "launch k_rel_join", e);
    }
    return 0;
}

}  // namespace

extern "C" {

const char* gvd_relattn_last_error(void) { return gvdd::g_err.c_str(); }

long long gvd_relattn_fwd_workspace(const gvd_relattn_problem* p)
{
    Geo g;
    const int rc = make_geo(p, g, "gvd_relattn_fwd_workspace");
    if (rc) return rc;
    const Plan pl = plan_of(g, p->B, compute_units());
    return pl.parts > 1 ? (long long)(part_rows(g, p->B, pl) * (64 * sizeof(float) + sizeof(float2))) : 0;
}

int gvd_relattn_fwd(const gvd_relattn_problem* p, const void* q, const void* k, const void* v, const void* table, void* out, float* lse,
                    void* workspace, void* stream)
{
    Geo g;
    const int rc = make_geo(p, g, "gvd_relattn_fwd");
    if (rc) return rc;
    if (!q || !k || !v || !table || !out) return fail(-1, "gvd_relattn_fwd: null pointer");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) return fail(-1, "gvd_relattn_fwd: pointers must be 16-byte aligned");
    g.table = table;
    return p->is_bf16 ? launch_fwd<__bf16>(g, p->B, q, k, v, out, lse, workspace, (hipStream_t)stream)
                      : launch_fwd<_Float16>(g, p->B, q, k, v, out, lse, workspace, (hipStream_t)stream);
}

}  // extern "C"
