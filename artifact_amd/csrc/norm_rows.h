// Layer norm of feature rows, forward and backward, with the ReLU and the dropout that may follow it in the same pass.
// Instantiated by norm_<input type>_<output type>.hip; the C ABI is in row_ops.hip.
//
// Of each row x (f columns), with w and b the parameters:
//     m = sum(x) / f      v = sum((x - m)^2) / f      r = 1 / sqrt(v + eps)      h = (x - m) r
//     pre = h w + b       y = D(max(pre, 0))          D: dropout, see philox_words; both are optional
// and of its gradient, with d = the gradient of y where D keeps the element, scaled like it, and pre > 0, else 0:
//     g = d w             dx = r (g - sum(g) / f - h sum(g h) / f)      dw = sum over rows of d h      db = ... of d
//
// A row is held in registers from its one read to its one write, so the variance is the mean square of the differences
// from the mean (no cancellation) at the price of one more cross-lane sum.  The backward pass keeps nothing from the
// forward one but x itself: statistics, gate and mask are computed again, which costs fewer bytes than storing them.
// Every launch is bounded by memory: 8 (forward) to 25 (backward) operations an element against 8 to 12 bytes of it.
#ifndef ROF_NORM_ROWS_H_
#define ROF_NORM_ROWS_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "rof.h"
#include "rof_internal.h"
#include "row_ops.h"

namespace rofn {

// ---- cross-lane sums ------------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }

struct Pair { int a, b; };
// {the other half's lanes beside one's own}, for rows of 16 lanes and for halves of 32
__device__ __forceinline__ Pair swap16(int v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {(int)r[0], (int)r[1]};
}
__device__ __forceinline__ Pair swap32(int v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {(int)r[0], (int)r[1]};
}

// The sum over the LPR lanes of a lane group, in every one of them: a butterfly of vector instructions only (lane pairs
// and quads by quad_perm, 8 and 16 lanes by mirrors, which meet a lane of the other half, 32 and 64 by the row swaps).
// Every step adds the same two numbers in both lanes, so all lanes hold the same bits.
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
    if (LPR > 1) v += __int_as_float(dpp<0xB1>(__float_as_int(v)));
    if (LPR > 2) v += __int_as_float(dpp<0x4E>(__float_as_int(v)));
    if (LPR > 4) v += __int_as_float(dpp<0x141>(__float_as_int(v)));
    if (LPR > 8) v += __int_as_float(dpp<0x140>(__float_as_int(v)));
    if (LPR > 16) {
        const Pair p = swap16(__float_as_int(v));
        v = __int_as_float(p.a) + __int_as_float(p.b);
    }
    if (LPR > 32) {
        const Pair p = swap32(__float_as_int(v));
        v = __int_as_float(p.a) + __int_as_float(p.b);
    }
    return v;
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    return __hiloint2double(dpp<CTRL>(__double2hiint(v)), dpp<CTRL>(__double2loint(v)));
}
template <int LPR>
__device__ __forceinline__ double group_sum(double v) {
    if (LPR > 1) v += dpp64<0xB1>(v);
    if (LPR > 2) v += dpp64<0x4E>(v);
    if (LPR > 4) v += dpp64<0x141>(v);
    if (LPR > 8) v += dpp64<0x140>(v);
    if (LPR > 16) {
        const Pair h = swap16(__double2hiint(v)), l = swap16(__double2loint(v));
        v = __hiloint2double(h.a, l.a) + __hiloint2double(h.b, l.b);
    }
    if (LPR > 32) {
        const Pair h = swap32(__double2hiint(v)), l = swap32(__double2loint(v));
        v = __hiloint2double(h.a, l.a) + __hiloint2double(h.b, l.b);
    }
    return v;
}

// ---- one row, spread over WAVES wavefronts of LPR lanes, K vectors of V columns per lane --------------------------
// Vector j of lane l (0 .. LPR * WAVES - 1) covers the columns (j * LPR * WAVES + l) * V and the next V - 1, so that one
// load instruction reads one contiguous piece of the row.  K is the least that covers f (checked by the launcher):
// every vector but a lane's last is whole.
template <typename TX, int LPR, int WAVES, int K>
struct RowMap {
    static constexpr int V = 16 / (int)sizeof(TX);
    static constexpr int LANES = LPR * WAVES;
    static constexpr int THREADS = WAVES > 4 ? WAVES * 64 : 256;
    static constexpr int ROWS = THREADS / LANES;      // rows a workgroup works on at a time
    static_assert(LPR == 64 || WAVES == 1, "a row is either part of a wavefront or whole wavefronts");

    int l;         // lane within the row
    int slot;      // which of the workgroup's rows
    int last;      // columns of the last vector that exist (0 .. V)

    __device__ __forceinline__ explicit RowMap(int f) {
        l = (int)threadIdx.x % LANES;
        slot = (int)threadIdx.x / LANES;
        const int left = f - col(K - 1);
        last = left < 0 ? 0 : left > V ? V : left;
    }
    __device__ __forceinline__ int col(int j) const { return (j * LANES + l) * V; }
    __device__ __forceinline__ bool has(int j, int e) const { return j < K - 1 || e < last; }

    // columns that do not exist read as zero, and so does everything when !ok
    template <typename T>
    __device__ __forceinline__ void load(const T *row, bool ok, float (&v)[K][V]) const {
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] = 0.f;
            if (!ok) continue;
            if (j < K - 1 || last == V) {
                load_vec<T, V>(row + col(j), v[j]);
            } else if (last > 0) {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < last) v[j][e] = load_one(row + col(j) + e);
            }
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T *row, const float (&v)[K][V]) const {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (j < K - 1 || last == V) {
                store_vec<T, V>(row + col(j), v[j]);
            } else if (last > 0) {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < last) store_one(row + col(j) + e, v[j][e]);
            }
        }
    }

    // Sum over the row's lanes.  Of several wavefronts: through `part`, which holds two sets of WAVES numbers and is used
    // alternately (`turn`), so that one barrier per sum is enough: a set is written again only after every wavefront has
    // passed the next sum's barrier, that is, has read it.
    template <typename S>
    __device__ __forceinline__ S sum(S v, S (*part)[WAVES], int &turn) const {
        v = group_sum<LPR>(v);
        if constexpr (WAVES > 1) {
            S *p = part[turn];
            turn ^= 1;
            if (l % 64 == 0) p[l / 64] = v;
            __syncthreads();
            v = S(0);
#pragma unroll
            for (int i = 0; i < WAVES; ++i) v += p[i];
        }
        return v;
    }

    // bit e of word j: whether the dropout keeps element (j, e).  A vector is a whole group of eight columns or half of one.
    __device__ __forceinline__ void kept(const Drop &d, int64_t row, int f, uint32_t (&bits)[K]) const {
        const uint64_t first = (uint64_t)row * (uint32_t)((f + 7) / 8);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            uint32_t w[4];
            philox_words(first + (uint32_t)(col(j) / 8), d, w);
            bits[j] = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const uint32_t word = V == 4 && (col(j) & 4) ? w[(2 + e / 2) % 4] : w[e / 2];
                const uint32_t u = e % 2 ? word >> 16 : word & 0xffffu;
                bits[j] |= (u >= d.threshold ? 1u : 0u) << e;
            }
        }
    }
};

// s / f from the reciprocal, with what the product leaves of s added: a row of equal numbers (a node without in-edges under
// a constant bias) has exactly that number as its mean, and no spread, where r = 1 / sqrt(eps) would magnify one rounding.
__device__ __forceinline__ float mean_of(float s, float f, float inv_f) {
    const float m = s * inv_f;
    return fmaf(fmaf(-m, f, s), inv_f, m);
}

template <int WAVES>
struct Scratch {
    float part[2][WAVES];
    double part64[2][WAVES];
};

template <typename TX, typename TY, int LPR, int WAVES, int K>
__global__ __launch_bounds__((RowMap<TX, LPR, WAVES, K>::THREADS)) void norm_fwd_kernel(NormArgs a) {
    using Map = RowMap<TX, LPR, WAVES, K>;
    constexpr int V = Map::V;
    __shared__ Scratch<WAVES> sh;
    const Map m(a.f);
    int turn = 0;
    float w[K][V], b[K][V];
    m.load(a.weight, a.weight != nullptr, w);
    m.load(a.bias, a.bias != nullptr, b);
    if (!a.weight) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) w[j][e] = 1.f;
    }
    const Drop drop(a);
    const float inv_f = 1.0f / (float)a.f;
    for (int64_t base = (int64_t)blockIdx.x * Map::ROWS; base < a.n; base += (int64_t)gridDim.x * Map::ROWS) {
        const int64_t row = base + m.slot;
        const bool ok = row < a.n;
        float v[K][V];
        m.load((const TX *)a.x + row * a.ldx, ok, v);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[j][e];
        const float mean = mean_of(m.sum(s, sh.part, turn), (float)a.f, inv_f);
        s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[j][e] = m.has(j, e) ? v[j][e] - mean : 0.f;
                s = fmaf(v[j][e], v[j][e], s);
            }
        const float r = 1.0f / sqrtf(m.sum(s, sh.part, turn) * inv_f + (float)a.eps);
        uint32_t bits[K];
        if (a.drop) m.kept(drop, row, a.f, bits);
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float y = fmaf(v[j][e] * r, w[j][e], b[j][e]);
                if (a.relu) y = y < 0.f ? 0.f : y;   // a NaN stays one
                if (a.drop) y = (bits[j] >> e & 1u) ? y * drop.scale : 0.f;
                v[j][e] = y;
            }
        if (ok) m.store((TY *)a.out + row * a.ldo, v);
    }
}

// The ReLU's gate decides whether a whole gradient passes, so its border must not move with the order in which a variant
// of this kernel adds.  Where |pre| is within the rounding error that 32 bits can have there, the wavefront (or the
// workgroup that shares the row) takes the row's statistics again in 64 bits and decides by those.  The bound, in half
// steps u = 2^-24: a lane adds up to 32 numbers, the butterfly and the wavefronts 6 + 16 more, so m is off by q / r with
// q = 55 u (|m| r + 1); h by q + 34 u |h| + |h| q^2 / 2, and the last operation adds 2 u (|h w| + |b|).  With |m| r up to
// 2^10 the square is below q, and all of it below 128 u = 2^-17 times |w| (r (|x| + |m|) + 1) + |b|; a row whose mean is
// further than that from zero is always decided in 64 bits.  About 2 elements in 10^5 are that close on normally
// distributed rows.
constexpr float kBorder = 7.62939453125e-06f;
constexpr float kFarMean = 1024.f;

template <typename TX, typename TY, int LPR, int WAVES, int K>
__global__ __launch_bounds__((RowMap<TX, LPR, WAVES, K>::THREADS)) void norm_bwd_kernel(NormArgs a) {
    using Map = RowMap<TX, LPR, WAVES, K>;
    constexpr int V = Map::V;
    __shared__ Scratch<WAVES> sh;
    const Map m(a.f);
    int turn = 0, turn64 = 0;
    float w[K][V], b[K][V], dw[K][V], db[K][V];
    m.load(a.weight, a.weight != nullptr, w);
    m.load(a.bias, a.bias != nullptr && a.relu, b);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (!a.weight) w[j][e] = 1.f;
            dw[j][e] = db[j][e] = 0.f;
        }
    const Drop drop(a);
    const float inv_f = 1.0f / (float)a.f;
    for (int64_t base = (int64_t)blockIdx.x * Map::ROWS; base < a.n; base += (int64_t)gridDim.x * Map::ROWS) {
        const int64_t row = base + m.slot;
        const bool ok = row < a.n;
        float x[K][V], d[K][V];
        m.load((const TX *)a.x + row * a.ldx, ok, x);
        m.load((const TY *)a.dout + row * a.ldd, ok, d);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) s += x[j][e];
        const float mean = mean_of(m.sum(s, sh.part, turn), (float)a.f, inv_f);
        s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float c = m.has(j, e) ? x[j][e] - mean : 0.f;
                s = fmaf(c, c, s);
            }
        const float r = 1.0f / sqrtf(m.sum(s, sh.part, turn) * inv_f + (float)a.eps);
        if (a.drop || a.relu) {
            uint32_t bits[K];   // the elements whose gradient passes
#pragma unroll
            for (int j = 0; j < K; ++j) bits[j] = 0xffu;
            if (a.drop) m.kept(drop, row, a.f, bits);
            if (a.relu) {
                uint32_t gate[K];
                bool near = r * fabsf(mean) > kFarMean;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    gate[j] = 0;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float pre = fmaf((x[j][e] - mean) * r, w[j][e], b[j][e]);
                        const float most = fmaf(fabsf(w[j][e]), fmaf(r, fabsf(x[j][e]) + fabsf(mean), 1.f), fabsf(b[j][e]));
                        near |= m.has(j, e) && (bits[j] >> e & 1u) && fabsf(pre) <= kBorder * most;
                        gate[j] |= (pre > 0.f ? 1u : 0u) << e;
                    }
                }
                near = near && ok;
                if (WAVES > 1 ? __syncthreads_or(near) : __any(near)) {
                    double s64 = 0.0;
#pragma unroll
                    for (int j = 0; j < K; ++j)
#pragma unroll
                        for (int e = 0; e < V; ++e) s64 += (double)x[j][e];
                    const double m64 = m.sum(s64, sh.part64, turn64) / a.f;
                    s64 = 0.0;
#pragma unroll
                    for (int j = 0; j < K; ++j)
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const double c = m.has(j, e) ? (double)x[j][e] - m64 : 0.0;
                            s64 = fma(c, c, s64);
                        }
                    const double r64 = 1.0 / sqrt(m.sum(s64, sh.part64, turn64) / a.f + a.eps);
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        gate[j] = 0;
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const double h = ((double)x[j][e] - m64) * r64;
                            gate[j] |= (fma(h, (double)w[j][e], (double)b[j][e]) > 0.0 ? 1u : 0u) << e;
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < K; ++j) bits[j] &= gate[j];
            }
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) d[j][e] = (bits[j] >> e & 1u) ? d[j][e] * drop.scale : 0.f;
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float h = m.has(j, e) ? (x[j][e] - mean) * r : 0.f;
                dw[j][e] = fmaf(d[j][e], h, dw[j][e]);
                db[j][e] += d[j][e];
                const float g = d[j][e] * w[j][e];
                s1 += g;
                s2 = fmaf(g, h, s2);
                x[j][e] = h;
                d[j][e] = g;
            }
        s1 = m.sum(s1, sh.part, turn) * inv_f;
        s2 = m.sum(s2, sh.part, turn) * inv_f;
        if (a.out) {
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) d[j][e] = r * (d[j][e] - s1 - x[j][e] * s2);
            if (ok) m.store((TX *)a.out + row * a.ldo, d);
        }
    }
    if (!a.partial) return;
    // The workgroup's sums, as one row of 2 f floats: lane groups of a wavefront first, then the wavefronts one after the
    // other through LDS (a fixed order).
    float *const pw = a.partial + (int64_t)blockIdx.x * 2 * a.f, *const pb = pw + a.f;
    if constexpr (WAVES > 1) {
        m.store(pw, dw);
        m.store(pb, db);
    } else {
        __shared__ float red[2 * LPR * K * V];
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int o = LPR; o < 64; o *= 2) {
                    dw[j][e] += __shfl_xor(dw[j][e], o);
                    db[j][e] += __shfl_xor(db[j][e], o);
                }
        for (int wave = 0; wave < 4; ++wave) {
            if ((int)threadIdx.x / 64 == wave && (int)threadIdx.x % 64 < LPR) {
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float *const at = red + m.col(j) + e;
                        at[0] = (wave ? at[0] : 0.f) + dw[j][e];
                        at[LPR * K * V] = (wave ? at[LPR * K * V] : 0.f) + db[j][e];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.f; c += 256) {
            pw[c] = red[c];
            pb[c] = red[LPR * K * V + c];
        }
    }
}

// ---- launch ---------------------------------------------------------------------------------------------------------
template <typename TX, typename TY, int LPR, int WAVES, int K>
int launch_variant(const NormArgs &a, bool backward, int blocks, hipStream_t st) {
    using Map = RowMap<TX, LPR, WAVES, K>;
    if (backward)
        hipLaunchKernelGGL((norm_bwd_kernel<TX, TY, LPR, WAVES, K>), dim3(blocks), dim3(Map::THREADS), 0, st, a);
    else
        hipLaunchKernelGGL((norm_fwd_kernel<TX, TY, LPR, WAVES, K>), dim3(blocks), dim3(Map::THREADS), 0, st, a);
    HIP_TRY(hipGetLastError());
    return ROF_OK;
}

// the variants that norm_shape (row_ops.hip) chooses among
template <typename TX, typename TY>
int launch_norm(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st) {
#define ROF_NORM_VARIANT(LPR, WAVES, K) \
    if (s.lpr == LPR && s.waves == WAVES && s.k == K) return launch_variant<TX, TY, LPR, WAVES, K>(a, backward, blocks, st)
    ROF_NORM_VARIANT(64, 1, 1);
    ROF_NORM_VARIANT(64, 1, 2);
    ROF_NORM_VARIANT(64, 1, 3);
    ROF_NORM_VARIANT(64, 1, 4);
    ROF_NORM_VARIANT(64, 4, 2);
    ROF_NORM_VARIANT(64, 4, 3);
    ROF_NORM_VARIANT(64, 4, 4);
    ROF_NORM_VARIANT(64, 16, 2);
    if constexpr (sizeof(TX) == 4) {   // 16384 bfloat16 columns are 2048 vectors
        ROF_NORM_VARIANT(64, 16, 3);
        ROF_NORM_VARIANT(64, 16, 4);
    }
#undef ROF_NORM_VARIANT
    return ROF_ERR_UNSUPPORTED;
}

}  // namespace rofn

#endif
