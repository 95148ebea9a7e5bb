// relattn_common.h -- shared by relattn_forward.hip and relattn_backward.hip: the bias by distance, the geometry of a call.
#pragma once
#include "../../include/gvd_relattn.h"
#include "diffusion_common.h"

namespace gvdr {

using namespace gvdd;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -3.4028234e38f;   // the running maximum before a row has seen anything: below every score that is not -infinity

// What every kernel of a call reads.  `first` by value: a few hundred bytes of kernel arguments, nothing on the device to keep or to upload.
struct Geo {
    int H, Nq, Nk, buckets, side, both, causal, reach, q_start, table_type;
    float scale, c, inv_scale;             // c = scale log2(e)
    const int* q_starts;
    const int* kv_lens;
    const void* table;
    long long q_bs, q_rs, kv_bs, kv_rs, o_bs, o_rs;
    int first[GVD_RELATTN_MAX_SIDE];
};

// The bias by distance lies in LDS for distances -reach - PAD .. reach + PAD: a block of 64 keys x 32 queries spans 95 distances, so a block with one
// distance inside (-reach, reach) reads no further.  Blocks without one have a single bias.
constexpr int PAD = 95;
__host__ __device__ inline int bias_len(int reach) { return 2 * (reach + PAD) + 1; }

__device__ __forceinline__ int bucket_of(const Geo& g, int d)
{
    const int n = g.both ? (d < 0 ? -d : d) : (d < 0 ? -d : 0);
    int b = -1;
    for (int k0 = 0; k0 < g.side; k0 += 16)   // (beyond side: the largest number)
#pragma unroll
        for (int k = 0; k < 16; k++) b += g.first[k0 + k] <= n;
    return b + (g.both && d > 0 ? g.side : 0);
}

__device__ __forceinline__ float table_at(const Geo& g, int bucket, int h)
{
    const int i = bucket * g.H + h;
    if (g.table_type == 0) return ((const float*)g.table)[i];
    if (g.table_type == 1) return (float)((const _Float16*)g.table)[i];
    return (float)((const __bf16*)g.table)[i];
}

// The bias as the products' accumulators start from it: over the scale, so that scores come out of the matrix unit as (q.k + bias / scale).  Entries at or below
// -10000 mask their bucket, as -infinity does: among them are the lowest values of every type and the constants used in their place, and a score that
// far out would leave 32 bits nothing for q.k.  For the same reason an entry counts as 10000 at most.
constexpr float MASKS_AT = -10000.f, MOST = 10000.f;
__device__ __forceinline__ float start_value(const Geo& g, float bias)
{
    return (bias <= MASKS_AT ? -INFINITY : (bias > MOST ? MOST : bias)) * g.inv_scale;
}

// Whether results do not depend on an entry: where it masks its bucket, and where another value counts in its place.
__device__ __forceinline__ bool without_gradient(float bias) { return bias <= MASKS_AT || bias > MOST; }

// MIRRORED: descending distances, for blocks whose registers run over queries.  Returns whether one of the lane's distances is masked.
template <bool MIRRORED = false>
__device__ __forceinline__ bool fill_bias(const Geo& g, int h, float* sBias, int tid, int nt)
{
    bool masked = false;
    for (int e = tid; e < bias_len(g.reach); e += nt) {
        const float x = start_value(g, table_at(g, bucket_of(g, MIRRORED ? g.reach + PAD - e : e - g.reach - PAD), h));
        masked |= x == -INFINITY;
        sBias[e] = x;
    }
    return masked;
}

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }
// (of a batch entry that is the same over a wave: held in scalar registers, so that loops and branches on them are scalar)
__device__ __forceinline__ int len_of(const Geo& g, int b) { return g.kv_lens ? __builtin_amdgcn_readfirstlane(clamp_int(g.kv_lens[b], 0, g.Nk)) : g.Nk; }
__device__ __forceinline__ int start_of(const Geo& g, int b) { return __builtin_amdgcn_readfirstlane(clamp_int(g.q_starts ? g.q_starts[b] : g.q_start, -(1 << 29), 1 << 29)); }

// A product's result as the next product's operand.  Of a 32 x 32 block a lane of half hi holds rows 4 hi + {0 .. 3, 8 .. 11, 16 .. 19, 24 .. 27} of one column, in registers'
// order; the matrix unit wants eight of the contraction's indexes a lane and step of 16, WHICH ones is free as long as both operands agree.  So the block goes on as it
// lies, registers 8 k2 .. + 7 packed, and the other operand brings rows 4 hi + {0 .. 3, 8 .. 11} of each 16: nothing is exchanged between the halves (that
// took 8 instructions a block).
template <typename T>
__device__ __forceinline__ typename Tr<T>::vec8 packed_operand(const unsigned (&pk)[8], int k2)
{
    typedef unsigned u4_ __attribute__((ext_vector_type(4)));
    const u4_ x = { pk[4 * k2], pk[4 * k2 + 1], pk[4 * k2 + 2], pk[4 * k2 + 3] };
    return __builtin_bit_cast(typename Tr<T>::vec8, x);
}

// ... and that other operand from the TRANSPOSE of a row-major LDS tile: lane (m = lane & 31, hi) gets column c0 + m of rows k0 + 4 hi + {0 .. 3, 8 .. 11}.  One
// transposing read hands each lane of a group of 16 one column of 4 rows x 16 columns, if lane s of the group points at row s / 4, columns 4 (s % 4) .. + 3.
// (Writing tiles a second time, transposed, took 6 dword writes and 2 more loads a lane and tile.)
template <typename T>
__device__ __forceinline__ typename Tr<T>::vec8 transposed_operand(const T* tile, int pitch, int k0, int c0, int lane)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    const T* p = tile + (k0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * pitch + c0 + (lane & 16) + 4 * (lane & 3);
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 8 * pitch));
    return __builtin_bit_cast(typename Tr<T>::vec8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Between LDS writes of a wave and reads by its other lanes: LDS operations of a wave keep their order, so this only keeps the compiler's.
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Sum of two packed 16-bit values and acc in 32 bits: one instruction, and of the ROUNDED weights that the matrix unit multiplies.
template <typename T> __device__ __forceinline__ float add_pair(unsigned packed, float acc)
{
    typedef T T2 __attribute__((ext_vector_type(2)));
    const T2 ones = { (T)1.0f, (T)1.0f };
    if constexpr (std::is_same<T, _Float16>::value) return __builtin_amdgcn_fdot2(__builtin_bit_cast(T2, packed), ones, acc, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(T2, packed), ones, acc, false);
}

// Host side: checks a problem and fills a Geo (the table's pointer aside).
int make_geo(const gvd_relattn_problem* p, Geo& g, const char* who);
int compute_units();

}  // namespace gvdr
