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
    int64_t jump;            // rows from the last of a workgroup's adjacent rounds to its next round
    int32_t inner;           // adjacent rounds
    int32_t f;
    int32_t relu;
    int32_t drop;            // dropout on
    uint32_t threshold;
    float scale;
    const int64_t *state;    // device: seed, offset
    int64_t call;
    double eps;
};

// the variant of the layer-norm kernels for a width, see norm_shape
struct NormShape {
    int lpr, waves, k;       // lanes of a wavefront and wavefronts that share a row, vectors per lane
    bool stream;             // backward: streaming accesses
    int rows() const { return waves > 1 ? 1 : 256 / lpr; }   // that a workgroup works on at a time
};

#define ROF_NORM_TYPES(V) V(f32_f32) V(f32_bf16) V(bf16_f32) V(bf16_bf16)
#define ROF_NORM_DECLARE(T)                                                                          \
    int norm_fwd_##T(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st);             \
    int norm_bwd_##T(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st);             \
    int norm_bwd_relu_##T(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st);
ROF_NORM_TYPES(ROF_NORM_DECLARE)
#undef ROF_NORM_DECLARE

#if defined(__HIPCC__)
// The dropout of one launch: key and offset are read from the device, so a captured launch draws from whatever the state
// holds when it is replayed.
struct Drop {
    uint32_t k0 = 0, k1 = 0, o0 = 0, o1 = 0;
    uint32_t last;           // the largest 16-bit number that drops an element: threshold - 1
    template <typename Args>
    __device__ __forceinline__ explicit Drop(const Args &a) : last(a.threshold - 1) {
        if (a.state) {
            const uint64_t seed = (uint64_t)a.state[0], offset = (uint64_t)a.state[1] + (uint64_t)a.call;
            k0 = (uint32_t)seed;
            k1 = (uint32_t)(seed >> 32);
            o0 = (uint32_t)offset;
            o1 = (uint32_t)(offset >> 32);
        }
    }
};

// Whether the element of field e (0 .. 7) is kept.  One comparison each: 16 bits of the low half of a word, 32 bits for the
// high half, whose lower bits cannot change the outcome against a bound that ends in ones.
__device__ __forceinline__ bool drop_keeps(uint32_t word, int e, const Drop &d) {
    return e % 2 ? word > (d.last << 16 | 0xffffu) : (uint16_t)word > (uint16_t)d.last;
}

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

// The elements of a vector of V columns from `col` on that the dropout keeps; `group` is the row's first.  A vector is a whole
// group of eight columns or half of one: the half's words are chosen as values (an index into the array would put it into
// memory, and a kernel that has to place memory per lane starts by asking the host for its launch shape: 14 us).
template <int V>
__device__ __forceinline__ void drop_kept(const Drop &d, uint64_t group, uint32_t col, bool (&keep)[V]) {
    uint32_t w[4];
    philox_words(group + col / 8, d, w);
    if constexpr (V == 4) {
        const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];
        const bool upper = col & 4;
        w[0] = upper ? w2 : w0;
        w[1] = upper ? w3 : w1;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) keep[e] = drop_keeps(w[e / 2], e, d);
}

typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));

// rounded to nearest even, like every bfloat16 this library stores
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const f2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2_t));
}
// V elements of a row as they lie in memory, so that a row can be under way in as few registers as it has bytes.
// Rows start wherever their type's alignment allows (packed rows of 47 columns), and the accesses promise no more than
// that: gfx950 reads and writes 4, 8, 12 and 16 bytes at any address, each with one instruction.
template <typename T, int V>
struct Packed {
    static constexpr int WORDS = V * (int)sizeof(T) / 4, PIECE = WORDS < 4 ? WORDS : 4;
    typedef uint32_t piece_t __attribute__((ext_vector_type(PIECE), aligned(sizeof(T))));
    uint32_t w[WORDS];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0;
    }
    // STREAM: bypassing the caches' replacement, for matrices that they do not hold until somebody reads them again
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < WORDS; i += PIECE) {
            const piece_t *at = reinterpret_cast<const piece_t *>(p) + i / PIECE;
            const piece_t t = STREAM ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
            for (int k = 0; k < PIECE; ++k) w[i + k] = t[k];
        }
    }
    template <bool STREAM = false>
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < WORDS; i += PIECE) {
            piece_t t;
#pragma unroll
            for (int k = 0; k < PIECE; ++k) t[k] = w[i + k];
            piece_t *at = reinterpret_cast<piece_t *>(p) + i / PIECE;
            if (STREAM)
                __builtin_nontemporal_store(t, at);
            else
                *at = t;
        }
    }
    // Moves the elements `by` (less than V) places to the front; what comes in behind them is anything.
    __device__ __forceinline__ void shift(int by) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t bytes = (uint32_t)(by & 1) * 2;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = __builtin_amdgcn_alignbyte(w[i + 1 < WORDS ? i + 1 : i], w[i], bytes);
            by >>= 1;
        }
        shift_words<1>(by);
        shift_words<2>(by);
        shift_words<4>(by);
    }
    // The first `count` elements only, the others zero (a row shorter than a vector; no hot path).
    __device__ __forceinline__ void load_few(const T *p, int count) {
        clear();
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e < count) {
                T t;
                __builtin_memcpy(&t, p + e, sizeof(T));
                if constexpr (sizeof(T) == 4)
                    w[e] = __float_as_uint(t);
                else
                    w[e / 2] |= (uint32_t)t << (e % 2 * 16);
            }
        }
    }
    // The first `count` (less than V) elements only.  `count` is the same for the whole launch, so the choice among the
    // V - 1 sizes is a scalar branch, and a size is one or two instructions.
    template <int C = V - 1>
    __device__ __forceinline__ void store_part(T *p, int count) const {
        if (count == C)
            __builtin_memcpy(p, w, C * sizeof(T));
        else if constexpr (C > 1)
            store_part<C - 1>(p, count);
    }
    template <int STEP>
    __device__ __forceinline__ void shift_words(int by) {
#pragma unroll
        for (int i = 0; i + STEP < WORDS; ++i) {
            const uint32_t here = w[i], there = w[i + STEP];   // as values: a choice between addresses would need memory
            w[i] = (by & STEP) ? there : here;
        }
    }
    __device__ __forceinline__ void unpack(float (&v)[V]) const {
#pragma unroll
        for (int e = 0; e < V; ++e)
            v[e] = __uint_as_float(sizeof(T) == 4 ? w[e] : e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
    __device__ __forceinline__ void pack(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = __float_as_uint(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 2) w[e / 2] = bf16_pair(v[e], v[e + 1]);
        }
    }
};
#endif

}  // namespace rofn

#endif
