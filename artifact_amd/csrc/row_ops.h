// What the row operators (row_ops.hip) and the layer-norm kernels (norm_rows.h) share: the dropout's random numbers, the
// access to rows, and the launch arguments.
#ifndef ROF_ROW_OPS_H_
#define ROF_ROW_OPS_H_

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rofn {

typedef uint16_t bf16_t;   // the bits of a bfloat16

struct NormArgs {
    const void *x;
    const void *dout;        // backward only
    const float *weight, *bias;
    void *out;               // forward: y; backward: dx, or null
    float *partial;          // backward: [workgroups][2][f], or null
    int64_t ldx, ldd, ldo;
    int64_t n;
    int32_t f;
    int32_t relu;
    int32_t drop;            // dropout on
    uint32_t threshold;
    float scale;
    const int64_t *state;    // device: seed, offset
    int64_t call;
    double eps;
};

// lanes of a row, vectors per lane: the variant of the layer-norm kernels that covers f columns
struct NormShape {
    int lpr, waves, k;
    int rows;                // rows a workgroup works on at a time
};

int launch_norm_f32_f32(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st);
int launch_norm_f32_bf16(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st);
int launch_norm_bf16_f32(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st);
int launch_norm_bf16_bf16(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st);

#if defined(__HIPCC__)
// The dropout of one launch: key and offset are read from the device, so a captured launch draws from whatever the state
// holds when it is replayed.
struct Drop {
    uint32_t k0 = 0, k1 = 0, o0 = 0, o1 = 0, threshold;
    float scale;
    template <typename Args>
    __device__ __forceinline__ explicit Drop(const Args &a) : threshold(a.threshold), scale(a.scale) {
        if (a.state) {
            const uint64_t seed = (uint64_t)a.state[0], offset = (uint64_t)a.state[1] + (uint64_t)a.call;
            k0 = (uint32_t)seed;
            k1 = (uint32_t)(seed >> 32);
            o0 = (uint32_t)offset;
            o1 = (uint32_t)(offset >> 32);
        }
    }
};

// Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011: the
// least that passes BigCrush): the four words of the counter (group, offset) under the key.  A group is eight columns of
// a row, 16 bits of the words each: with 32 bits per element a bfloat16 pass would be bounded by the multiplications (14
// wide products per call), with 16 they hide behind the loads; the price is that a rate is a multiple of 2^-16.
__device__ __forceinline__ void philox_words(uint64_t group, const Drop &d, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = d.o0, c3 = d.o1, k0 = d.k0, k1 = d.k1;
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}

// Rows start wherever their type's alignment allows (packed rows of 47 columns): the vectors promise no more than that,
// and gfx950 reads and writes them with one instruction all the same.
typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const bf16_t *p) { return __uint_as_float((uint32_t)*p << 16); }
// rounded to nearest even, like every bfloat16 this library stores
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const f2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2_t));
}
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16_t *p, float v) { *p = (bf16_t)bf16_pair(v, 0.f); }

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const f4_t t = *reinterpret_cast<const f4_t *>(p + i);
            v[i] = t.x;
            v[i + 1] = t.y;
            v[i + 2] = t.z;
            v[i + 3] = t.w;
        }
    } else {
        uint32_t t[V / 2];
        if constexpr (V == 8) {
            const u4_t u = *reinterpret_cast<const u4_t *>(p);
            t[0] = u.x;
            t[1] = u.y;
            t[2] = u.z;
            t[3] = u.w;
        } else {
            const u2_t u = *reinterpret_cast<const u2_t *>(p);
            t[0] = u.x;
            t[1] = u.y;
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            v[2 * i] = __uint_as_float(t[i] << 16);
            v[2 * i + 1] = __uint_as_float(t[i] & 0xffff0000u);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            f4_t t;
            t.x = v[i];
            t.y = v[i + 1];
            t.z = v[i + 2];
            t.w = v[i + 3];
            *reinterpret_cast<f4_t *>(p + i) = t;
        }
    } else if constexpr (V == 8) {
        u4_t t;
        t.x = bf16_pair(v[0], v[1]);
        t.y = bf16_pair(v[2], v[3]);
        t.z = bf16_pair(v[4], v[5]);
        t.w = bf16_pair(v[6], v[7]);
        *reinterpret_cast<u4_t *>(p) = t;
    } else {
        u2_t t;
        t.x = bf16_pair(v[0], v[1]);
        t.y = bf16_pair(v[2], v[3]);
        *reinterpret_cast<u2_t *>(p) = t;
    }
}
#endif

}  // namespace rofn

#endif
