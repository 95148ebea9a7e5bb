// adamw.hip -- one AdamW step over many tensors at once for gfx950 (C-ABI: include/gvd_optim.h).
//
//     m' = m + (1 - b1) (g - m),  v' = b2 v + (1 - b2) g^2,  p' = keep p - step_size m' / (root_factor sqrt(v') + eps)
//
// Bound by memory: every element is read and written once -- 28 bytes with 32-bit moments and fp32 parameters, 16 with 8-bit ones -- and no
// element depends on another (with 8-bit moments: on its block of 256).  So: one launch for up to MAX_TENSORS tensors (their table travels in
// the kernel's arguments: nothing to upload, nothing that a captured graph could find changed), workgroups of CHUNK consecutive elements,
// 16-byte accesses.
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
constexpr int CHUNK = 2048;       // elements a workgroup: eight blocks of 8-bit moments, two rounds of 256 lanes x 4
constexpr int BLOCK = GVD_ADAMW_BLOCK;

struct Table {
    gvd_adamw_tensor t[MAX_TENSORS];
    unsigned first[MAX_TENSORS];   // first workgroup of each tensor, ascending
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

// Four consecutive elements as floats; beyond n: zeros.  `wide` (all pointers of the tensor aligned to a vector): one access where all four are there.
template <typename T>
__device__ __forceinline__ f4 load4(const T* __restrict__ p, long long i, long long n, bool wide)
{
    f4 r = { 0.f, 0.f, 0.f, 0.f };
    if (wide && i + 4 <= n) {
        const typename Vec4<T>::type x = *reinterpret_cast<const typename Vec4<T>::type*>(p + i);
#pragma unroll
        for (int j = 0; j < 4; j++) r[j] = (float)x[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) r[j] = (float)p[i + j];
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store4(T* __restrict__ p, long long i, long long n, bool wide, f4 v)
{
    if (wide && i + 4 <= n) {
        typename Vec4<T>::type x;
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (T)v[j];
        *reinterpret_cast<typename Vec4<T>::type*>(p + i) = x;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) p[i + j] = (T)v[j];
    }
}

__device__ __forceinline__ unsigned load4_bytes(const unsigned char* __restrict__ p, long long i, long long n, bool wide)
{
    if (wide && i + 4 <= n) return *reinterpret_cast<const unsigned*>(p + i);
    unsigned r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i + j < n) r |= (unsigned)p[i + j] << (8 * j);
    return r;
}

__device__ __forceinline__ void store4_bytes(unsigned char* __restrict__ p, long long i, long long n, bool wide, unsigned v)
{
    if (wide && i + 4 <= n) { *reinterpret_cast<unsigned*>(p + i) = v; return; }
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

// the tensor that workgroup `wg` belongs to: the last whose first workgroup is not behind it (uniform: scalar code)
__device__ __forceinline__ int tensor_of(const Table& a, unsigned wg)
{
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first[mid] <= wg) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(256) k_adamw32(const Table a, float w1, float b2, float w2, float eps, const void* __restrict__ scalars)
{
    const int k = tensor_of(a, blockIdx.x);
    const gvd_adamw_tensor& t = a.t[k];
    const Step st = step_of(a, k, scalars);
    T* __restrict__ p = (T*)t.param;
    const T* __restrict__ g = (const T*)t.grad;
    float* __restrict__ m = (float*)t.exp_avg;
    float* __restrict__ v = (float*)t.exp_avg_sq;
    const long long n = t.n, at = (long long)(blockIdx.x - a.first[k]) * CHUNK + 4 * threadIdx.x;
    const bool wide = (((uintptr_t)p | (uintptr_t)g) % (4 * sizeof(T)) | ((uintptr_t)m | (uintptr_t)v) % 16) == 0;
    constexpr int R = CHUNK / 1024;
    f4 pp[R], gg[R], mm[R], vv[R];
#pragma unroll
    for (int r = 0; r < R; r++) {   // all loads of the workgroup's chunk in flight at once
        const long long i = at + 1024 * r;
        gg[r] = load4(g, i, n, wide);
        mm[r] = load4(m, i, n, wide);
        vv[r] = load4(v, i, n, wide);
        pp[r] = load4(p, i, n, wide);
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
            pn[j] = st.keep * pp[r][j] - st.step_size * (mn[j] / (sqrtf(vn[j]) * st.root_factor + eps));
        }
        store4(m, i, n, wide, mn);
        store4(v, i, n, wide, vn);
        store4(p, i, n, wide, pn);
    }
}

// x in [0, 448] as e4m3, rounded up with the probability of its distance from the lower neighbour (u: 16 random bits).  Scaled by 2^-120 a float's own
// exponent and upper mantissa bits ARE the code, subnormals of the one becoming subnormals of the other; what is cut off is what the draw is added to.
// least: the code that a value above 0 has at least.  What is not finite becomes e4m3's NaN.
__device__ __forceinline__ unsigned to_e4m3(float x, unsigned u, unsigned least)
{
    const unsigned b = (__float_as_uint(fminf(x, 448.f) * 0x1p-120f) + (u << 4)) >> 20;
    const unsigned c = b < least ? least : (b > 0x7eu ? 0x7eu : b);
    return x < INFINITY ? c : 0x7fu;
}

__device__ __forceinline__ float wave_max(float x)
{
#pragma unroll
    for (int s = 32; s; s >>= 1) x = fmaxf(x, __shfl_xor(x, s, 64));
    return x;
}

// The largest finite magnitude of four values.
__device__ __forceinline__ float finite_max(f4 x)
{
    float r = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float y = fabsf(x[j]);
        r = y < INFINITY ? fmaxf(r, y) : r;   // (also skips NaN)
    }
    return r;
}

// A block whose largest magnitude is below this is held as zeros: 1 / big would overflow.  (A root is never that small unless it is 0: the least
// positive float's root is 3.7e-23.)
constexpr float TINY = 0x1p-110f;

template <typename T>
__global__ void __launch_bounds__(256) k_adamw8(const Table a, float w1, float b2, float w2, float eps, const void* __restrict__ scalars)
{
    const int k = tensor_of(a, blockIdx.x);
    const gvd_adamw_tensor& t = a.t[k];
    const Step st = step_of(a, k, scalars);
    T* __restrict__ p = (T*)t.param;
    const T* __restrict__ g = (const T*)t.grad;
    unsigned char* __restrict__ m8 = (unsigned char*)t.exp_avg;
    unsigned char* __restrict__ r8 = (unsigned char*)t.exp_avg_sq;
    float* __restrict__ ms = t.exp_avg_scale;
    float* __restrict__ rs = t.exp_avg_sq_scale;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long n = t.n, at = (long long)(blockIdx.x - a.first[k]) * CHUNK + BLOCK * wave;
    const bool wide = (((uintptr_t)p | (uintptr_t)g) % (4 * sizeof(T)) | ((uintptr_t)m8 | (uintptr_t)r8) % 4) == 0;
    constexpr int R = CHUNK / (4 * BLOCK);
    f4 pp[R], gg[R];
    unsigned mc[R], rc[R];
    float sm[R], sr[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const long long base = at + 4 * BLOCK * r, i = base + 4 * lane;
        gg[r] = load4(g, i, n, wide);
        mc[r] = load4_bytes(m8, i, n, wide);
        rc[r] = load4_bytes(r8, i, n, wide);
        pp[r] = load4(p, i, n, wide);
        sm[r] = base < n ? ms[base / BLOCK] : 0.f;
        sr[r] = base < n ? rs[base / BLOCK] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const long long base = at + 4 * BLOCK * r, i = base + 4 * lane;
        if (base >= n) continue;   // (uniform over the wave)
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
            pn[j] = st.keep * pp[r][j] - st.step_size * (mn[j] / (rn[j] * st.root_factor + eps));
        }
        store4(p, i, n, wide, pn);
        const float bm = wave_max(finite_max(mn)), br = wave_max(finite_max(rn));   // (elements beyond n: zeros)
        const float fm = bm >= TINY ? 1.f / bm * 448.f : 0.f, fr = br >= TINY ? 1.f / br * 448.f : 0.f;
        unsigned cm = 0, cr = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned h = mix((unsigned)(i + j) * 0x9D2C5681u + st.key);
            const unsigned c = to_e4m3(fabsf(mn[j]) * fm, h & 0xffffu, 0u);
            cm |= (c | (mn[j] < 0.f ? 0x80u : 0u)) << (8 * j);
            cr |= to_e4m3(rn[j] * fr, h >> 16, rn[j] > 0.f ? 1u : 0u) << (8 * j);
        }
        store4_bytes(m8, i, n, wide, cm);
        store4_bytes(r8, i, n, wide, cr);
        if (lane == 0) {
            ms[base / BLOCK] = bm >= TINY ? bm / 448.f : 0.f;
            rs[base / BLOCK] = br >= TINY ? br / 448.f : 0.f;
        }
    }
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
        if (t.n < 0 || t.n > (1LL << 40)) return fail(-1, "gvd_adamw_step: a tensor's size is out of range");
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
            if (wgs && wgs + more > 0x7fffffffULL) break;
            a.t[a.count] = tensors[i];
            a.first[a.count++] = (unsigned)wgs;
            wgs += more;
        }
        if (!wgs) continue;
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
