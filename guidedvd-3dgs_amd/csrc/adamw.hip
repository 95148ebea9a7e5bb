// adamw.hip -- one AdamW step over many tensors at once for gfx950 (C-ABI: include/gvd_optim.h).
//
//     m' = m + (1 - b1) (g - m),  v' = b2 v + (1 - b2) g^2,  p' = keep p - step_size m' / (root_factor sqrt(v') + eps)
//
// Bound by memory: every element is read and written once -- 28 bytes with 32-bit moments and fp32 parameters, 16 with 8-bit ones -- and no
// element depends on another (with 8-bit moments: on its block of 256).  So: one launch for up to MAX_TENSORS tensors (their table travels in
// the kernel's arguments: nothing to upload, nothing that a captured graph could find changed), workgroups of CHUNK consecutive elements,
// 16-byte accesses.  118M fp32 elements: 560 us, 5.9 TB/s (a plain copy of that size reaches 4.9); 11.8M with 8-bit moments: 33 us, 5.7 TB/s.
//
// 8-bit moments.  m and r = sqrt(v) are held as e4m3 (4 significant bits, 2^-9 .. 448) with one scale a block of 256 consecutive elements
// (largest magnitude / 448), a block per wave.  Two choices carry this:
//   * the ROOT is held: its range is half of v's in powers of two, and r is what the update divides by;
//   * rounding is stochastic: a step moves v by (1 - b2) = 0.1 % of itself, far below half of e4m3's distance of 1/16 .. 1/8, so nearest rounding would
//     leave every value where it is for ever; rounded up with the probability of its distance from the lower neighbour the running mean stays
//     unbiased.  The draw is a hash of (seed, tensor, step, element): the same run gives the same result.
//   * r > 0 is never held as 0: it would make the next update divide by eps alone.
// m', v', p' of this step use the unrounded values.  Products and sums are rounded one by one (no contraction): the moments, and with them the codes that
// the draws pick, are bit for bit those of the same formulas as elementwise operations.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <string>

#include "../../include/gvd_optim.h"

namespace {

thread_local std::string g_err;
int fail(int code, const char* what, hipError_t e = hipSuccess)
{
    char buf[384];
    if (e != hipSuccess) snprintf(buf, sizeof buf, "%s: %s", what, hipGetErrorString(e));
    else snprintf(buf, sizeof buf, "%s", what);
    g_err = buf;
    return code;
}

constexpr int MAX_TENSORS = 52;   // 52 * 76 bytes and the other arguments: below 4 KiB of kernel arguments
constexpr int CHUNK = 2048;       // elements a workgroup: eight blocks of 8-bit moments, two rounds of 256 lanes x 4 (11.8M elements with 8-bit moments, ordinary accesses: 37.1 us; 1024 37.5, 4096 42.6)
constexpr int BLOCK = GVD_ADAMW_BLOCK;
constexpr long long MOST_WORKGROUPS = GVD_ADAMW_MOST / CHUNK;   // of a launch: 2^23, 2^31 lanes

struct Table {
    gvd_adamw_tensor t[MAX_TENSORS];
    unsigned first[MAX_TENSORS];   // first workgroup of each tensor, ascending; unused entries: the largest number
    int count;
};

__host__ __device__ inline unsigned mix(unsigned h)
{
    h = (h ^ (h >> 16)) * 0x7A2D4F2Du;
    h = (h ^ (h >> 15)) * 0x5C8B3B55u;
    return h ^ (h >> 16);
}

__host__ __device__ inline unsigned make_key(unsigned seed, unsigned tensor, unsigned step)
{
    return mix(mix(mix(seed + 0x3D1C27A5u) ^ tensor) ^ step);
}

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef f4 type; };
template <> struct Vec4<_Float16> { typedef h4 type; };
template <> struct Vec4<__bf16> { typedef b4 type; };

// Four consecutive elements as floats.  FULL: all of the workgroup's elements are there and every pointer is aligned to a vector; otherwise one by one,
// zeros beyond n.  (Chosen once a workgroup, so the code of a full one has no branch around an access.)  Nothing is read twice: non-temporal accesses, 562 us
// for 118M elements against 615 with ordinary ones (603 with the loads alone, 613 with the stores alone).
template <bool FULL, typename T>
__device__ __forceinline__ f4 load4(const T* __restrict__ p, long long i, long long n)
{
    f4 r = { 0.f, 0.f, 0.f, 0.f };
    if (FULL) {
        const typename Vec4<T>::type x = __builtin_nontemporal_load(reinterpret_cast<const typename Vec4<T>::type*>(p + i));
#pragma unroll
        for (int j = 0; j < 4; j++) r[j] = (float)x[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) r[j] = (float)p[i + j];
    }
    return r;
}

template <bool FULL, typename T>
__device__ __forceinline__ void store4(T* __restrict__ p, long long i, long long n, f4 v)
{
    if (FULL) {
        typename Vec4<T>::type x;
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (T)v[j];
        __builtin_nontemporal_store(x, reinterpret_cast<typename Vec4<T>::type*>(p + i));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) p[i + j] = (T)v[j];
    }
}

template <bool FULL>
__device__ __forceinline__ unsigned load4_bytes(const unsigned char* __restrict__ p, long long i, long long n)
{
    if (FULL) return *reinterpret_cast<const unsigned*>(p + i);
    unsigned r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i + j < n) r |= (unsigned)p[i + j] << (8 * j);
    return r;
}

template <bool FULL>
__device__ __forceinline__ void store4_bytes(unsigned char* __restrict__ p, long long i, long long n, unsigned v)
{
    if (FULL) { *reinterpret_cast<unsigned*>(p + i) = v; return; }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i + j < n) p[i + j] = (unsigned char)(v >> (8 * j));
}

struct Step { float step_size, root_factor, keep; unsigned key; };

__device__ __forceinline__ Step step_of(const Table& a, int k, const void* scalars)
{
    if (scalars) {
        const float* s = reinterpret_cast<const float*>(scalars) + 4 * k;
        return { s[0], s[1], s[2], __float_as_uint(s[3]) };
    }
    return { a.t[k].step_size, a.t[k].root_factor, a.t[k].keep, a.t[k].key };
}

// The tensor that workgroup `wg` belongs to: the last whose first workgroup is not behind it.  All entries are compared (scalar code; unused ones are the
// largest number): one trip to memory for the table, where a binary search makes one for each of its steps.
__device__ __forceinline__ int tensor_of(const Table& a, unsigned wg)
{
    int k = -1;
#pragma unroll
    for (int i = 0; i < MAX_TENSORS; i++) k += a.first[i] <= wg;
    return k;
}

// p' from m', sqrt(v') and the step: the reciprocal is the unit's own (1 ulp), 2^-23 of an update.
__device__ __forceinline__ float new_param(const Step& st, float p, float m, float root, float eps)
{
    return st.keep * p - st.step_size * (m * __builtin_amdgcn_rcpf(root * st.root_factor + eps));
}

template <typename T, bool FULL>
__device__ __forceinline__ void chunk32(const gvd_adamw_tensor& t, const Step& st, long long at, float w1, float b2, float w2, float eps)
{
    T* __restrict__ p = (T*)t.param;
    const T* __restrict__ g = (const T*)t.grad;
    float* __restrict__ m = (float*)t.exp_avg;
    float* __restrict__ v = (float*)t.exp_avg_sq;
    const long long n = t.n;
    constexpr int R = CHUNK / 1024;
    f4 pp[R], gg[R], mm[R], vv[R];
#pragma unroll
    for (int r = 0; r < R; r++) {   // all loads of the workgroup's chunk in flight at once
        const long long i = at + 1024 * r;
        gg[r] = load4<FULL>(g, i, n);
        mm[r] = load4<FULL>(m, i, n);
        vv[r] = load4<FULL>(v, i, n);
        pp[r] = load4<FULL>(p, i, n);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const long long i = at + 1024 * r;
        f4 pn, mn, vn;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float gj = gg[r][j];
            mn[j] = mm[r][j] + w1 * (gj - mm[r][j]);
            vn[j] = b2 * vv[r][j] + w2 * (gj * gj);
            pn[j] = new_param(st, pp[r][j], mn[j], sqrtf(vn[j]), eps);
        }
        store4<FULL>(m, i, n, mn);
        store4<FULL>(v, i, n, vn);
        store4<FULL>(p, i, n, pn);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_adamw32(const Table a, float w1, float b2, float w2, float eps, const void* __restrict__ scalars)
{
    const int k = tensor_of(a, blockIdx.x);
    const gvd_adamw_tensor& t = a.t[k];
    const Step st = step_of(a, k, scalars);
    const long long begin = (long long)(blockIdx.x - a.first[k]) * CHUNK, at = begin + 4 * threadIdx.x;
    const bool wide = (((uintptr_t)t.param | (uintptr_t)t.grad) % (4 * sizeof(T)) | ((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) % 16) == 0;
    if (wide && begin + CHUNK <= t.n) chunk32<T, true>(t, st, at, w1, b2, w2, eps);
    else chunk32<T, false>(t, st, at, w1, b2, w2, eps);
}

// x in [0, 448] as e4m3, rounded up with the probability of its distance from the lower neighbour (u: 16 random bits at 4 .. 19).  Scaled by 2^-120 a float's
// own exponent and upper mantissa bits ARE the code, subnormals of the one becoming subnormals of the other; what is cut off is what the draw is added
// to, and 448 plus a draw is still 448: also where the product that made x was rounded up, by 15 steps at most.
__device__ __forceinline__ unsigned to_e4m3(float x, unsigned u) { return (__float_as_uint(x * 0x1p-120f) + u) >> 20; }

// The largest of the wave's values, in all lanes (scalar): over rows of 16, then across the rows, without LDS.
__device__ __forceinline__ unsigned wave_max(unsigned x)
{
#define GVD_STEP(ctrl, rows) { const unsigned y = __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false); x = x > y ? x : y; }
    GVD_STEP(0x111, 0xf)   // row_shr:1
    GVD_STEP(0x112, 0xf)   // row_shr:2
    GVD_STEP(0x114, 0xf)   // row_shr:4
    GVD_STEP(0x118, 0xf)   // row_shr:8
    GVD_STEP(0x142, 0xa)   // row_bcast:15 into rows 1 and 3
    GVD_STEP(0x143, 0xc)   // row_bcast:31 into rows 2 and 3
#undef GVD_STEP
    return __builtin_amdgcn_readlane(x, 63);
}

// Largest magnitude of a block as a float's bits (for values >= 0 they order as the values do); what is not finite lies above all that is.
constexpr unsigned MAGNITUDE = 0x7fffffffu, NOT_FINITE = 0x7f800000u;
__device__ __forceinline__ unsigned largest(f4 x, bool finite_only)
{
    unsigned r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const unsigned y = __float_as_uint(x[j]) & MAGNITUDE;
        if (!finite_only || y < NOT_FINITE) r = r > y ? r : y;
    }
    return wave_max(r);
}

// A block whose largest magnitude is below this is held as zeros: 1 / big would overflow.  (A root is never that small unless it is 0: the least positive
// float's root is 3.7e-23.)
constexpr float TINY = 0x1p-110f;

template <typename T, bool FULL>
__device__ __forceinline__ void chunk8(const gvd_adamw_tensor& t, const Step& st, long long at, int lane, float w1, float b2, float w2, float eps)
{
    T* __restrict__ p = (T*)t.param;
    const T* __restrict__ g = (const T*)t.grad;
    unsigned char* __restrict__ m8 = (unsigned char*)t.exp_avg;
    unsigned char* __restrict__ r8 = (unsigned char*)t.exp_avg_sq;
    float* __restrict__ ms = t.exp_avg_scale;
    float* __restrict__ rs = t.exp_avg_sq_scale;
    const long long n = t.n;
    constexpr int R = CHUNK / (4 * BLOCK);
    f4 pp[R], gg[R];
    unsigned mc[R], rc[R];
    float sm[R], sr[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const long long base = at + 4 * BLOCK * r, i = base + 4 * lane;
        gg[r] = load4<FULL>(g, i, n);
        mc[r] = load4_bytes<FULL>(m8, i, n);
        rc[r] = load4_bytes<FULL>(r8, i, n);
        pp[r] = load4<FULL>(p, i, n);
        sm[r] = FULL || base < n ? ms[base / BLOCK] : 0.f;
        sr[r] = FULL || base < n ? rs[base / BLOCK] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const long long base = at + 4 * BLOCK * r, i = base + 4 * lane;
        if (!FULL && base >= n) continue;   // (uniform over the wave)
        const f4 m0 = { __builtin_amdgcn_cvt_f32_fp8(mc[r], 0), __builtin_amdgcn_cvt_f32_fp8(mc[r], 1),
                        __builtin_amdgcn_cvt_f32_fp8(mc[r], 2), __builtin_amdgcn_cvt_f32_fp8(mc[r], 3) };
        const f4 r0 = { __builtin_amdgcn_cvt_f32_fp8(rc[r], 0), __builtin_amdgcn_cvt_f32_fp8(rc[r], 1),
                        __builtin_amdgcn_cvt_f32_fp8(rc[r], 2), __builtin_amdgcn_cvt_f32_fp8(rc[r], 3) };
        f4 pn, mn, rn;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float gj = gg[r][j], mj = m0[j] * sm[r], rj = r0[j] * sr[r];
            mn[j] = mj + w1 * (gj - mj);
            rn[j] = sqrtf(b2 * (rj * rj) + w2 * (gj * gj));
            pn[j] = new_param(st, pp[r][j], mn[j], rn[j], eps);
        }
        store4<FULL>(p, i, n, pn);
        unsigned bm = largest(mn, false), br = largest(rn, false);   // (elements beyond n: zeros)
        const bool odd = bm >= NOT_FINITE || br >= NOT_FINITE;
        if (odd) { bm = largest(mn, true); br = largest(rn, true); }
        // both scales at once: the moment's in the even lanes, the root's in the odd ones
        const float big = __uint_as_float(lane & 1 ? br : bm);
        const float scale = big >= TINY ? big * (1.f / 448.f) : 0.f, times = big >= TINY ? 1.f / big * 448.f : 0.f;
        const float fm = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(times), 0)), fr = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(times), 1));
        unsigned cm = 0, cr = 0;
        const unsigned h0 = (unsigned)i * 0x9D2C5681u + st.key;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned h = mix(h0 + j * 0x9D2C5681u), least = min(__float_as_uint(rn[j]), 1u);   // (a root above 0 has code 1 at least)
            const unsigned c = to_e4m3(fabsf(mn[j]) * fm, (h << 4) & 0xffff0u), d = to_e4m3(rn[j] * fr, (h >> 12) & 0xffff0u);
            cm |= (c | ((__float_as_uint(mn[j]) >> 24) & 0x80u)) << (8 * j);
            cr |= max(d, least) << (8 * j);
        }
        if (odd) {   // (uniform) what is not finite is held as e4m3's NaN; its code above is arbitrary, in more bits than its own 8: all four anew
            cm = cr = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned h = mix(h0 + j * 0x9D2C5681u), least = min(__float_as_uint(rn[j]), 1u);
                unsigned c = to_e4m3(fabsf(mn[j]) * fm, (h << 4) & 0xffff0u), d = to_e4m3(rn[j] * fr, (h >> 12) & 0xffff0u);
                d = max(d, least);
                if ((__float_as_uint(mn[j]) & MAGNITUDE) >= NOT_FINITE) c = 0x7fu;
                if ((__float_as_uint(rn[j]) & MAGNITUDE) >= NOT_FINITE) d = 0x7fu;
                cm |= (c | ((__float_as_uint(mn[j]) >> 24) & 0x80u)) << (8 * j);
                cr |= d << (8 * j);
            }
        }
        store4_bytes<FULL>(m8, i, n, cm);
        store4_bytes<FULL>(r8, i, n, cr);
        if (lane < 2) (lane ? rs : ms)[base / BLOCK] = scale;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_adamw8(const Table a, float w1, float b2, float w2, float eps, const void* __restrict__ scalars)
{
    const int k = tensor_of(a, blockIdx.x);
    const gvd_adamw_tensor& t = a.t[k];
    const Step st = step_of(a, k, scalars);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long begin = (long long)(blockIdx.x - a.first[k]) * CHUNK, at = begin + BLOCK * wave;
    const bool wide = (((uintptr_t)t.param | (uintptr_t)t.grad) % (4 * sizeof(T)) | ((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) % 4) == 0;
    if (wide && begin + CHUNK <= t.n) chunk8<T, true>(t, st, at, lane, w1, b2, w2, eps);
    else chunk8<T, false>(t, st, at, lane, w1, b2, w2, eps);
}

struct Counters {
    float* step[MAX_TENSORS];
    const float* lr_at[MAX_TENSORS];
    double lr[MAX_TENSORS], wd[MAX_TENSORS];
    unsigned id[MAX_TENSORS];
    int count;
};

// one lane a tensor: counts the step and makes its scalars (64 bits, as the host does)
__global__ void __launch_bounds__(64) k_adamw_scalars(const Counters a, double b1, double b2, unsigned seed, float* __restrict__ scalars)
{
    const int k = threadIdx.x;
    if (k >= a.count) return;
    const float t = *a.step[k] + 1.f;
    *a.step[k] = t;
    const double lr = a.lr_at[k] ? (double)*a.lr_at[k] : a.lr[k];
    scalars[4 * k] = (float)(lr / (1.0 - pow(b1, (double)t)));
    scalars[4 * k + 1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    scalars[4 * k + 2] = (float)(1.0 - lr * a.wd[k]);
    scalars[4 * k + 3] = __uint_as_float(make_key(seed, a.id[k], (unsigned)t));
}

bool bad_betas(double b1, double b2) { return !(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0); }

}  // namespace

extern "C" {

const char* gvd_optim_last_error(void) { return g_err.c_str(); }

unsigned gvd_adamw_key(unsigned seed, unsigned tensor, unsigned step) { return make_key(seed, tensor, step); }

int gvd_adamw_step(const gvd_adamw_tensor* tensors, int count, int param_type, int state_bits, double beta1, double beta2, double eps,
                   const void* scalars, void* stream_)
{
    if (count < 0 || (count && !tensors)) return fail(-1, "gvd_adamw_step: bad arguments");
    if (param_type < 0 || param_type > 2) return fail(-1, "gvd_adamw_step: param_type must be 0 (float), 1 (fp16) or 2 (bf16)");
    if (state_bits != 8 && state_bits != 32) return fail(-1, "gvd_adamw_step: state_bits must be 8 or 32");
    if (bad_betas(beta1, beta2) || !(eps >= 0.0)) return fail(-1, "gvd_adamw_step: betas must be in [0, 1) and eps at least 0");
    for (int i = 0; i < count; i++) {
        const gvd_adamw_tensor& t = tensors[i];
        if (t.n < 0 || t.n > GVD_ADAMW_MOST) return fail(-1, "gvd_adamw_step: a tensor's size is out of range");
        if (t.n && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale))))
            return fail(-1, "gvd_adamw_step: a tensor has a null pointer");
    }
    hipStream_t stream = (hipStream_t)stream_;
    const float w1 = (float)(1.0 - beta1), b2 = (float)beta2, w2 = (float)(1.0 - beta2), e = (float)eps;
    for (int i = 0; i < count;) {
        Table a;
        a.count = 0;
        unsigned long long wgs = 0;
        const int from = i;
        for (; i < count && a.count < MAX_TENSORS; i++) {
            const unsigned long long more = (unsigned long long)((tensors[i].n + CHUNK - 1) / CHUNK);
            if (wgs && wgs + more > (unsigned long long)MOST_WORKGROUPS) break;
            a.t[a.count] = tensors[i];
            a.first[a.count++] = (unsigned)wgs;
            wgs += more;
        }
        if (!wgs) continue;
        for (int j = a.count; j < MAX_TENSORS; j++) a.first[j] = 0xffffffffu;
        const void* sc = scalars ? (const char*)scalars + 16 * (size_t)from : nullptr;
        const dim3 grid((unsigned)wgs);
#define GVD_LAUNCH(K, T) hipLaunchKernelGGL(K<T>, grid, dim3(256), 0, stream, a, w1, b2, w2, e, sc)
        if (state_bits == 32) {
            if (param_type == 0) GVD_LAUNCH(k_adamw32, float); else if (param_type == 1) GVD_LAUNCH(k_adamw32, _Float16); else GVD_LAUNCH(k_adamw32, __bf16);
        } else {
            if (param_type == 0) GVD_LAUNCH(k_adamw8, float); else if (param_type == 1) GVD_LAUNCH(k_adamw8, _Float16); else GVD_LAUNCH(k_adamw8, __bf16);
        }
#undef GVD_LAUNCH
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return fail(-2, "launch k_adamw", err);
    }
    return 0;
}

int gvd_adamw_scalars(float* const* steps, const float* const* lrs, const double* lr, const double* weight_decay, const unsigned* tensor_ids,
                      int count, double beta1, double beta2, unsigned seed, void* scalars, void* stream_)
{
    if (count < 0 || (count && (!steps || !lr || !weight_decay || !tensor_ids || !scalars))) return fail(-1, "gvd_adamw_scalars: bad arguments");
    if (bad_betas(beta1, beta2)) return fail(-1, "gvd_adamw_scalars: betas must be in [0, 1)");
    for (int i = 0; i < count; i++)
        if (!steps[i]) return fail(-1, "gvd_adamw_scalars: a step is a null pointer");
    for (int from = 0; from < count; from += MAX_TENSORS) {
        Counters a;
        a.count = count - from < MAX_TENSORS ? count - from : MAX_TENSORS;
        for (int i = 0; i < a.count; i++) {
            a.step[i] = steps[from + i];
            a.lr_at[i] = lrs ? lrs[from + i] : nullptr;
            a.lr[i] = lr[from + i];
            a.wd[i] = weight_decay[from + i];
            a.id[i] = tensor_ids[from + i];
        }
        hipLaunchKernelGGL(k_adamw_scalars, dim3(1), dim3(64), 0, (hipStream_t)stream_, a, beta1, beta2, seed, (float*)scalars + 4 * (size_t)from);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return fail(-2, "launch k_adamw_scalars", err);
    }
    return 0;
}

}  // extern "C"
