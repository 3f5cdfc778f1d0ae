// Layer norm of feature rows, forward and backward, with the ReLU and the dropout that may follow it in the same pass.
// Instantiated by norm_fwd_<input type>_<output type>.hip and norm_bwd_...; the C ABI is in row_ops.hip.
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
// An element is 8 (forward) to 25 (backward) operations, with dropout a quarter or an eighth of a generator's call more (14
// wide products and twice as many other operations), against 8 and 12 bytes of float32 rows or 4 and 6 of bfloat16 ones.
// Rows that are part of a wavefront are bounded by memory in either type; those of several wavefronts, and of several
// bfloat16 vectors per lane, by what their registers leave of wavefronts to hide the barriers and the loads behind.
//
// Times in this header and in row_ops.hip are of the kernel alone, events around twenty launches; figures that are compared
// are of one run, and runs differ by up to 5 %.  A profiler's are up to 10 % longer.
#ifndef ROF_NORM_ROWS_H_
#define ROF_NORM_ROWS_H_

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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

// The sum of a lane's N numbers as a balanced tree: as many additions as in a row, but each number passes ceil(log2 N).
template <int N>
__device__ __forceinline__ float tree_sum(const float *v) {
    if constexpr (N == 1)
        return v[0];
    else
        return tree_sum<(N + 1) / 2>(v) + tree_sum<N / 2>(v + (N + 1) / 2);
}

// s / f from the reciprocal, with what the product leaves of s added: a row of equal numbers (a node without in-edges under
// a constant bias) has exactly that number as its mean, and no spread, where r = 1 / sqrt(eps) would magnify one rounding.
__device__ __forceinline__ float mean_of(float s, float f, float inv_f) {
    const float m = s * inv_f;
    return fmaf(fmaf(-m, f, s), inv_f, m);
}

// ---- one row, spread over WAVES wavefronts of LPR lanes, K vectors of V columns per lane --------------------------
// Vector j of lane l (0 .. LPR * WAVES - 1) covers the columns (j * LPR * WAVES + l) * V and the next V - 1, so that one
// load instruction reads one contiguous piece of the row.  K is the least that covers f (checked by the launcher):
// every vector but a lane's last is whole.
template <typename TX, int LPR, int WAVES, int K>
struct RowMap {
    static constexpr int V = 16 / (int)sizeof(TX);
    static constexpr int LANES = LPR * WAVES, WAVES_ = WAVES, K_ = K;
    static constexpr int THREADS = WAVES > 1 ? WAVES * 64 : 256;
    static constexpr int ROWS = THREADS / LANES;      // rows a workgroup works on at a time
    static_assert(LPR == 64 || WAVES == 1, "a row is either part of a wavefront or whole wavefronts");
    static_assert(WAVES == 1 || ROWS == 1, "the sums of several wavefronts meet in LDS that is there once per workgroup");

    int l;         // lane within the row
    int slot;      // which of the workgroup's rows
    int last;      // columns of the last vector that exist (0 .. V)
    int tail;      // f % V: what `last` is in the one lane where it is neither 0 nor V
    bool full;     // the row fills all lanes' vectors: nothing below has to ask which columns exist
    int from;      // column at which the last vector is read
    int back;      // how far before its own columns that is (V - tail; 0 in lanes with whole vectors)
    float columns, inv_columns;   // of the lane's wavefront, and 1 / columns (0 if it has none)

    __device__ __forceinline__ explicit RowMap(int f) {
        l = (int)threadIdx.x % LANES;
        slot = (int)threadIdx.x / LANES;
        tail = f % V;
        full = f == LANES * K * V;
        const int left = f - col(K - 1);
        last = left < 0 ? 0 : left > V ? V : left;
        from = last == V ? col(K - 1) : f - V;
        back = last > 0 ? V - last : 0;
        columns = columns_of(f, l / 64);
        inv_columns = columns > 0.f ? 1.0f / columns : 0.f;
    }
    // the columns that wavefront i of the row covers
    static __device__ __forceinline__ float columns_of(int f, int i) {
        const int left = f - ((K - 1) * LANES + i * 64) * V, most = 64 * V;
        return (float)((K - 1) * most + (left < 0 ? 0 : left > most ? most : left));
    }
    __device__ __forceinline__ int col(int j) const { return (j * LANES + l) * V; }
    __device__ __forceinline__ bool has(int j, int e) const { return j < K - 1 || e < last; }

    // A lane's part of a row as it lies in memory.  Nothing is branched around: a load whose result meets another value at a
    // join is waited for there, and the next row's could not stay under way.  So a lane without columns reads the row's last
    // V, and so does the last vector of a row that is no multiple of V, which is shifted into place when it is unpacked
    // (element by element, rows of 47 columns took 1.4 times as long as rows of 48, bfloat16 2.6 times).  Only a row shorter
    // than one vector is read element by element.
    template <typename T>
    struct Part {
        Packed<T, V> p[K];
        template <bool STREAM>
        __device__ __forceinline__ void load(const RowMap &m, const T *row) {
#pragma unroll
            for (int j = 0; j < K - 1; ++j) p[j].template load<STREAM>(row + m.col(j));
            if constexpr (LANES == 1)
                p[K - 1].load_few(row, m.last);
            else
                p[K - 1].template load<STREAM>(row + m.from);
        }
        // Waits for the row here.  Placed before this row's stores: the counter that a load is waited for by is in order, so
        // a wait after them would be one for the stores as well.
        __device__ __forceinline__ void arrive() {
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int i = 0; i < Packed<T, V>::WORDS; ++i) asm volatile("" : "+v"(p[j].w[i]));
        }
        // columns that do not exist are anything
        __device__ __forceinline__ void unpack(const RowMap &m, float (&v)[K][V]) {
            if (LANES > 1 && m.tail) p[K - 1].shift(m.back);
#pragma unroll
            for (int j = 0; j < K; ++j) p[j].unpack(v[j]);
        }
    };
    // a parameter's columns: `none` without a parameter, `missing` where there is no column
    __device__ __forceinline__ void load_param(const float *q, float none, float missing, float (&v)[K][V]) const {
        Part<float> t;
        if (q) {
            t.template load<false>(*this, q);
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) t.p[j].clear();
        }
        t.unpack(*this, v);
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (!q) v[j][e] = none;
                if (!has(j, e)) v[j][e] = missing;
            }
    }
    template <bool STREAM, typename T>
    __device__ __forceinline__ void store(T *row, const float (&v)[K][V]) const {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            Packed<T, V> p;
            p.pack(v[j]);
            if (j < K - 1 || last == V)
                p.template store<STREAM>(row + col(j));
            else if (last > 0)
                p.store_part(row + col(j), tail);
        }
    }

    // Two sums over the row's lanes.  Of several wavefronts: through `part`, which holds two sets and is used alternately
    // (`turn`), so that one barrier is enough: a set is written again only after every wavefront has passed the next one's
    // barrier, that is, has read it.
    template <typename S>
    __device__ __forceinline__ void sum2(S &v0, S &v1, S (*part)[WAVES][2], int &turn) const {
        v0 = group_sum<LPR>(v0);
        v1 = group_sum<LPR>(v1);
        if constexpr (WAVES > 1) {
            S(*p)[2] = part[turn];
            turn ^= 1;
            if (l % 64 == 0) {
                p[l / 64][0] = v0;
                p[l / 64][1] = v1;
            }
            __syncthreads();
            v0 = v1 = S(0);
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                v0 += p[i][0];
                v1 += p[i][1];
            }
        }
    }

    // Mean of a row's elements and the sum of the squares of their differences from it; v becomes the differences (0 where
    // there is no column).  Of several wavefronts each takes its own columns' first, and the row's follow from theirs: the
    // squares are theirs plus (columns) (their mean - the mean)^2, one barrier for both.  `apart`: how far the mean of the
    // wavefront's columns is from the row's.
    __device__ __forceinline__ void moments(float (&v)[K][V], float f, float inv_f, float (*part)[WAVES][2], int &turn, float &mean,
                                            float &squares, float &apart) const {
        if (!full) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[K - 1][e] = has(K - 1, e) ? v[K - 1][e] : 0.f;
        }
        float s = group_sum<LPR>(tree_sum<K * V>(&v[0][0]));
        float own = WAVES > 1 ? mean_of(s, columns, inv_columns) : mean_of(s, f, inv_f);   // columns: the wavefront's
        subtract(v, own);
        constexpr int CHAINS = K * V < 8 ? 2 : 4;   // of K V / CHAINS products each
        float c[CHAINS];
#pragma unroll
        for (int i = 0; i < K * V; ++i) {
            const float d = v[i / V][i % V];
            c[i % CHAINS] = i < CHAINS ? d * d : fmaf(d, d, c[i % CHAINS]);
        }
        float q = group_sum<LPR>(tree_sum<CHAINS>(c));
        apart = 0.f;
        if constexpr (WAVES > 1) {
            float(*p)[2] = part[turn];
            turn ^= 1;
            if (l % 64 == 0) {
                p[l / 64][0] = own;
                p[l / 64][1] = q;
            }
            __syncthreads();
            const float first = own;
            s = q = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) s = fmaf(columns_of((int)f, i), p[i][0], s);
            own = mean_of(s, f, inv_f);
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                const float d = p[i][0] - own;
                q += fmaf(columns_of((int)f, i) * d, d, p[i][1]);
            }
            apart = fabsf(own - first);
            subtract(v, own - first);
        }
        mean = own;
        squares = q;
    }
    __device__ __forceinline__ void subtract(float (&v)[K][V], float from) const {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] -= from;
        if (!full) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[K - 1][e] = has(K - 1, e) ? v[K - 1][e] : 0.f;
        }
    }
};

// The rounds of a workgroup: `inner` of them next to each other, then the same again a whole launch further on.
struct Rounds {
    int64_t left;      // rows from this round's first one to the matrix's end
    int64_t step;      // rows from this round to the next
    int32_t in;
    template <int ROWS>
    __device__ __forceinline__ static int64_t first(const NormArgs &a) { return (int64_t)blockIdx.x * a.inner * ROWS; }
    __device__ __forceinline__ Rounds(const NormArgs &a, int64_t first, int rows) : left(a.n - first), in(a.inner) { plan(a, rows); }
    __device__ __forceinline__ void plan(const NormArgs &a, int rows) { step = in == 1 ? a.jump : rows; }
    __device__ __forceinline__ void next(const NormArgs &a, int rows) {
        left -= step;
        in = in == 1 ? a.inner : in - 1;
        plan(a, rows);
    }
};

// Where a lane's row begins, from one round to the next; it stays on its last row when the next would be behind the matrix.
// `all` (the same in every lane): no lane of the workgroup is that far, which spares the choice.
template <typename T>
struct Cursor {
    T *at;
    int64_t ld;
    __device__ __forceinline__ Cursor(T *base, int64_t ld_, int64_t row, int64_t rows)
        : at(base + (row < rows ? row : rows - 1) * ld_), ld(ld_) {}
    __device__ __forceinline__ void advance(int64_t step, bool all, bool further) {
        if (all || further) at += step * ld;
    }
};

__device__ __forceinline__ float relu_of(float v) { return __builtin_elementwise_maximum(v, 0.f); }   // a NaN stays one

template <int WAVES>
struct Scratch {
    float part[2][WAVES][2];
    double part64[2][WAVES][2];
};

// A lane's columns of a parameter.  In registers, but in LDS in the backward kernel of rows that are several wavefronts:
// there a lane holds up to 32 columns, and it is registers (of the gradient's sums above all) that bound the wavefronts in
// flight (20011 x 4099 bfloat16 with ReLU and dropout: 210 us with them in registers, 141 from LDS; without ReLU no
// difference, and the forward kernel, which has registers to spare, 2 to 10 % slower from LDS).  A lane reads back only what it
// wrote, 16 bytes at a time in lane order, so there is neither a barrier nor a conflict.
template <typename Map, bool BACKWARD>
struct Param {
    static constexpr bool kLds = BACKWARD && Map::WAVES_ > 1;
    static constexpr int V = Map::V, K = Map::K_, Q = V / 4;
    using Store = float4[kLds ? K * Q * Map::LANES : 1];
    float v[kLds ? 1 : K][V];
    float4 *lds;

    __device__ __forceinline__ Param(const Map &m, const float *q, float none, float missing, Store &store, float &most,
                                     float factor = 1.f) {
        float t[K][V];
        m.load_param(q, none, missing, t);
        most = 0.f;
        lds = store + (kLds ? m.l : 0);
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (m.has(j, e)) most = fmaxf(most, fabsf(t[j][e]));
                t[j][e] *= factor;
            }
            set(j, t[j]);
        }
    }
    // For a bias of which only the sign of h w + bias matters, as in the backward kernel: where the weight is zero that is the
    // bias's own sign, which an infinity has as well.  Such a column is then never near the border, where one with a weight and
    // a bias of zero would take every row through the 64-bit statistics (2^22 x 256 bfloat16 with ReLU and dropout and one such
    // column: 1955 us, without it 1124).
    template <typename W>
    __device__ __forceinline__ void decide(const W &weight) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float w[V], b[V];
            weight.get(j, w);
            get(j, b);
#pragma unroll
            for (int e = 0; e < V; ++e) b[e] = w[e] != 0.f ? b[e] : b[e] > 0.f ? __builtin_inff() : -__builtin_inff();
            set(j, b);
        }
    }
    __device__ __forceinline__ void set(int j, const float (&from)[V]) {
        if constexpr (kLds) {
#pragma unroll
            for (int i = 0; i < Q; ++i)
                lds[(j * Q + i) * Map::LANES] = make_float4(from[4 * i], from[4 * i + 1], from[4 * i + 2], from[4 * i + 3]);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] = from[e];
        }
    }
    __device__ __forceinline__ void get(int j, float (&to)[V]) const {
        if constexpr (kLds) {
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float4 t = lds[(j * Q + i) * Map::LANES];
                to[4 * i] = t.x;
                to[4 * i + 1] = t.y;
                to[4 * i + 2] = t.z;
                to[4 * i + 3] = t.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) to[e] = v[j][e];
        }
    }
};

// Forward.  A lane group works on one row while its next one is on its way; reads and writes the matrix once.  Of the bytes
// it moves: 2^18 x 256 float32 96 us, 5.6 TB/s, with ReLU 97; 2.4 M x 47 float32 182 us, 5.0; 2^20 x 128 bfloat16 to float32
// 165 us, 4.9; 20011 x 4099 bfloat16 73 us, 4.5; with ReLU and dropout 10^6 x 100 float32 150 us, 5.3; 2^22 x 256 bfloat16
// 740 us, 5.8 (a copy reaches 4.5 to 5.9); 16384 x 16 float32 4 us, which is a launch.
template <typename TX, typename TY, int LPR, int WAVES, int K>
__global__ __launch_bounds__((RowMap<TX, LPR, WAVES, K>::THREADS)) void norm_fwd_kernel(NormArgs a) {
    using Map = RowMap<TX, LPR, WAVES, K>;
    constexpr int V = Map::V;
    __shared__ Scratch<WAVES> sh;
    const Map m(a.f);
    int turn = 0;
    __shared__ typename Param<Map, false>::Store wstore, bstore;
    float most;
    // the dropout's scale is in the parameters: it is positive, so it passes through the ReLU
    const Param<Map, false> weight(m, a.weight, 1.f, 0.f, wstore, most, a.scale), bias(m, a.bias, 0.f, 0.f, bstore, most, a.scale);
    const float f = (float)a.f, inv_f = 1.0f / f, eps = (float)a.eps;
    const int64_t first = Rounds::first<Map::ROWS>(a);
    Rounds go(a, first, Map::ROWS);
    const uint32_t groups = (uint32_t)(a.f + 7) / 8;
    typename Map::template Part<TX> next;
    const int64_t row = first + m.slot;
    uint64_t group = (uint64_t)row * groups;
    Cursor<const TX> x((const TX *)a.x, a.ldx, row, a.n);
    Cursor<TY> out((TY *)a.out, a.ldo, row, a.n);
    next.template load<false>(m, x.at);
    const Drop drop(a);   // read from memory: after the first row is on its way
    for (; go.left > 0; go.next(a, Map::ROWS)) {
        const bool ok = m.slot < go.left, all = go.step + Map::ROWS <= go.left, further = m.slot + go.step < go.left;
        float v[K][V];
        next.unpack(m, v);
        x.advance(go.step, all, further);
        next.template load<false>(m, x.at);   // on its way while this row is worked on
        float mean, squares, apart;
        m.moments(v, f, inv_f, sh.part, turn, mean, squares, apart);
        const float r = rsqrtf(fmaf(squares, inv_f, eps));
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float w[V], b[V];
            weight.get(j, w);
            bias.get(j, b);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[j][e] = fmaf(v[j][e] * r, w[e], b[e]);
                if (a.relu) v[j][e] = relu_of(v[j][e]);
            }
            if (a.drop) {
                bool keep[V];
                drop_kept(drop, group, (uint32_t)m.col(j), keep);
#pragma unroll
                for (int e = 0; e < V; ++e) v[j][e] = keep[e] ? v[j][e] : 0.f;
            }
        }
        next.arrive();
        if (ok) m.template store<false>(out.at, v);
        out.advance(go.step, all, further);
        group += (uint64_t)go.step * groups;
    }
}

// The ReLU's gate decides whether a whole gradient passes, so its border must not move with the order in which a variant
// of this kernel adds.  Where |pre| is within the rounding error that 32 bits can have there, the wavefront (or the
// workgroup that shares the row) takes the row's statistics again in 64 bits and decides by those.  The bound, in half
// steps u = 2^-24, with F = |m| r + 1, which mean|x| r is at most, for a row of one wavefront or less:
//   m: 5 additions in a lane, 6 across, 2 for the division: 13 u of mean|x|, so h is off by q = 13 u F;
//   the squares: 2 u from the differences, 8 in a lane, 6 across: 16 u, so r by 8 u, by 3 u from its own operations (the sum
//   with eps, the root), and by q^2 / 2 from m, which is 6 u for |m| r up to kFarMean; h by 2 u more: 19 u |h|.  Near the
//   border |h w| is |b|, and the last operation adds 2 u |b|: in all 13 u F |w| + 21 u |b|.
// For several wavefronts:
//   m: 10 u more (eight weighted means, 2 for the division): 23 u F;  the difference is taken in two steps, off by u of
//   its wavefront's mean's distance from m (`apart`) twice, and by u |h| once more;
//   the squares: 2 u more in a lane, 12 u for the wavefronts', so r by 15 + 3 + 17 u; and the error e of a wavefront's
//   mean counts once with that mean's distance from m: 2 e (distance) (columns) summed over the wavefronts is at most
//   2 * 13 u F of the squares (Cauchy and Schwarz), r by 13 u F: 38 u |h| + 13 u F |h|;  in all 23 u F |w| + 2 u r (apart) |w| +
//   (40 + 13 F) u |b|.
// So 32 u and 64 u times F (|w| + |b|) + r (apart) |w|; for w and b a lane's largest serve, so that the common path has
// one minimum per element.  A row whose mean is further from zero than kFarMean / r is always decided in 64 bits.  About 4
// elements in 10^6 are that close on normally distributed rows, 8 in rows of several wavefronts.  (20011 x 4099 bfloat16 with
// ReLU and dropout: 141 us; 130 if none ever came here, 159 with a border of four times the width.)
template <int WAVES>
constexpr float kBorder = WAVES > 1 ? 3.814697265625e-06f : 1.9073486328125e-06f;
constexpr float kFarMean = 1024.f;

// The exact sign of pre, in place of its value.  Rare, so it is kept out of the registers of the common path: the row is read
// again, a vector at a time.  Not slow either: on a small graph one wavefront that comes here is what the launch waits for.
template <typename Map, typename TX, typename W, typename B>
__device__ __forceinline__ void gate64(const Map &m, const NormArgs &a, const TX *row, const W &weight, const B &bias,
                                       double (*part)[Map::WAVES_][2], int &turn, float (&pre)[Map::K_][Map::V]) {
    constexpr int V = Map::V, K = Map::K_;
    auto at = [&](int j, float (&v)[V]) {   // columns that do not exist are zero
        Packed<TX, V> p;
        if constexpr (Map::LANES == 1) {
            p.load_few(row, m.last);
        } else {
            p.load(row + (j < K - 1 ? m.col(j) : m.from));
            if (j == K - 1 && m.tail) p.shift(m.back);
        }
        p.unpack(v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = m.has(j, e) ? v[e] : 0.f;
    };
    float v[V];
    double s = 0.0, none = 0.0;
#pragma unroll 1
    for (int j = 0; j < K; ++j) {
        at(j, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s += (double)v[e];
    }
    m.sum2(s, none, part, turn);
    const double mean = s / a.f;
    s = none = 0.0;
#pragma unroll 1
    for (int j = 0; j < K; ++j) {
        at(j, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double c = m.has(j, e) ? (double)v[e] - mean : 0.0;
            s = fma(c, c, s);
        }
    }
    m.sum2(s, none, part, turn);
    const double r = 1.0 / sqrt(s / a.f + a.eps);
#pragma unroll
    for (int j = 0; j < K; ++j) {
        float w[V], b[V];
        at(j, v);
        weight.get(j, w);
        bias.get(j, b);
#pragma unroll
        for (int e = 0; e < V; ++e) pre[j][e] = fma(((double)v[e] - mean) * r, (double)w[e], (double)b[e]) > 0.0 ? 1.f : 0.f;
        asm volatile("" ::: "memory");   // one vector after the other
    }
}

// nothing, where the bias is not needed (without a ReLU the gradient does not depend on it)
struct NoParam {
    using Store = float4[1];
    template <typename Map>
    __device__ __forceinline__ NoParam(const Map &, const float *, float, float, Store &, float &) {}
};
template <typename Map, bool NEEDED>
using ParamOf = std::conditional_t<NEEDED, Param<Map, true>, NoParam>;

// Backward.  As forward, with the gradient's row beside that of x: two reads and a write, and the parameters' gradients of the
// workgroup's rows in registers up to its end.  Without the parameters' gradients (with
// them 6 to 13 us more): 2.4 M x 47 float32 247 us, 5.5 TB/s; 2^20 x 64 bfloat16 67 us, 6.0 (a third of it from the Infinity
// Cache); 20011 x 4099 bfloat16 107 us, 4.6 (six vectors in flight per lane are what its registers hold), with ReLU and dropout
// 137 us; with them also 10^6 x 100 float32 208 us, 5.8; 2^20 x 128 bfloat16 to float32 185 us, 5.8; 2^22 x 256 bfloat16
// 1119 us, 5.8; 16384 x 16 float32 4.2 us.
// Two rows ahead instead of one are no gain (2^22 x 256 bfloat16 1425 us, with one 1355, before the launch was cut into tiles).
template <typename TX, typename TY, int LPR, int WAVES, int K, bool RELU, bool STREAM>
__global__ __launch_bounds__((RowMap<TX, LPR, WAVES, K>::THREADS)) void norm_bwd_kernel(NormArgs a) {
    using Map = RowMap<TX, LPR, WAVES, K>;
    constexpr int V = Map::V;
    __shared__ Scratch<WAVES> sh;
    const Map m(a.f);
    int turn = 0, turn64 = 0;
    __shared__ typename Param<Map, true>::Store wstore;
    __shared__ typename ParamOf<Map, RELU>::Store bstore;
    float dw[K][V], db[K][V], wmost, bmost;
    const Param<Map, true> weight(m, a.weight, 1.f, 0.f, wstore, wmost);
    // in columns that do not exist pre is -infinity: never near the border, and the gate is closed
    ParamOf<Map, RELU> bias(m, a.bias, 0.f, -__builtin_inff(), bstore, bmost);
    if constexpr (RELU) bias.decide(weight);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[j][e] = db[j][e] = 0.f;
    const float f = (float)a.f, inv_f = 1.0f / f, eps = (float)a.eps;
    const int64_t first = Rounds::first<Map::ROWS>(a);
    Rounds go(a, first, Map::ROWS);
    const uint32_t groups = (uint32_t)(a.f + 7) / 8;
    typename Map::template Part<TX> next_x;
    typename Map::template Part<TY> next_d;
    const int64_t row = first + m.slot;
    uint64_t group = (uint64_t)row * groups;
    Cursor<const TX> x((const TX *)a.x, a.ldx, row, a.n);
    Cursor<const TY> dout((const TY *)a.dout, a.ldd, row, a.n);
    Cursor<TX> dx((TX *)a.out, a.ldo, row, a.n);
    next_x.template load<STREAM>(m, x.at);
    next_d.template load<STREAM>(m, dout.at);
    const Drop drop(a);   // read from memory: after the first row is on its way
    for (; go.left > 0; go.next(a, Map::ROWS)) {
        const bool ok = m.slot < go.left, all = go.step + Map::ROWS <= go.left, further = m.slot + go.step < go.left;
        float h[K][V], d[K][V];
        next_x.unpack(m, h);
        next_d.unpack(m, d);
        const TX *const here = x.at;
        x.advance(go.step, all, further);   // on their way while this row is worked on
        dout.advance(go.step, all, further);
        next_x.template load<STREAM>(m, x.at);
        next_d.template load<STREAM>(m, dout.at);
        // Columns that do not exist hold other columns of d.  Their weight is 0 and their sums are not stored, but an infinity
        // or a NaN that the dropout or the gate stops in its own column has to be stopped there as well, so both do.
        if (go.left < Map::ROWS) {   // lane groups behind the last row work on it once more and add nothing
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) d[j][e] = ok ? d[j][e] : 0.f;
        }
        float mean, squares, apart;
        m.moments(h, f, inv_f, sh.part, turn, mean, squares, apart);
        const float r = rsqrtf(fmaf(squares, inv_f, eps));
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) h[j][e] *= r;
        if (a.drop) {   // its scale comes last: everything below is linear in d
#pragma unroll
            for (int j = 0; j < K; ++j) {
                bool keep[V];
                drop_kept(drop, group, (uint32_t)m.col(j), keep);
#pragma unroll
                for (int e = 0; e < V; ++e) d[j][e] = keep[e] && (RELU || m.has(j, e)) ? d[j][e] : 0.f;
            }
        }
        if constexpr (RELU) {
            float pre[K][V], least = __builtin_inff();
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float w[V], b[V];
                weight.get(j, w);
                bias.get(j, b);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    pre[j][e] = fmaf(h[j][e], w[e], b[e]);
                    least = fminf(least, fabsf(pre[j][e]));
                }
            }
            const float far = r * fabsf(mean);
            const bool close = ok && (far > kFarMean || least <= kBorder<WAVES> * fmaf(far + 1.f, wmost + bmost, r * apart * wmost));
            if (WAVES > 1 ? __syncthreads_or(close) : __any(close)) gate64(m, a, here, weight, bias, sh.part64, turn64, pre);
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) d[j][e] = pre[j][e] > 0.f ? d[j][e] : 0.f;
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float w[V];
            weight.get(j, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                dw[j][e] = fmaf(d[j][e], h[j][e], dw[j][e]);
                db[j][e] += d[j][e];
                d[j][e] *= w[e];
                s1 += d[j][e];
                s2 = fmaf(d[j][e], h[j][e], s2);
            }
        }
        m.sum2(s1, s2, sh.part, turn);
        next_x.arrive();
        next_d.arrive();
        if (a.out) {
            const float rs = r * a.scale;
            s1 *= -inv_f * rs;
            s2 *= -inv_f * rs;
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) d[j][e] = fmaf(h[j][e], s2, fmaf(d[j][e], rs, s1));
            if (ok) m.template store<STREAM>(dx.at, d);
            dx.advance(go.step, all, further);
        }
        group += (uint64_t)go.step * groups;
    }
    if (!a.partial) return;
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            dw[j][e] *= a.scale;
            db[j][e] *= a.scale;
        }
    // The workgroup's sums, as one row of 2 f floats: lane groups of a wavefront first, then the wavefronts one after the
    // other through LDS (a fixed order).
    float *const pw = a.partial + (int64_t)blockIdx.x * 2 * a.f, *const pb = pw + a.f;
    if constexpr (WAVES > 1) {
        m.template store<false>(pw, dw);
        m.template store<false>(pb, db);
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
// The variants that norm_shape (row_ops.hip) chooses among: lanes of a wavefront, wavefronts and vectors per lane.
// (V(lanes, wavefronts, vectors); STREAMED: those that also exist with streaming accesses; F32, BF16: for rows of that type.)
#define ROF_NORM_STREAMED(V) V(8, 1, 1) V(16, 1, 1) V(32, 1, 1) V(64, 1, 1) V(64, 1, 2) V(64, 2, 2) V(64, 3, 2) V(64, 4, 2) V(64, 8, 2)
#define ROF_NORM_F32(V) V(8, 1, 2) V(16, 1, 2) V(32, 1, 2)
#define ROF_NORM_BF16(V) V(4, 1, 3) V(8, 1, 3) V(16, 1, 3)
#define ROF_NORM_OTHERS(V) V(1, 1, 1) V(2, 1, 1) V(4, 1, 1) V(32, 1, 3) V(64, 1, 3) V(64, 3, 3) V(64, 4, 3) V(64, 8, 3) V(64, 8, 4)

template <typename TX, typename TY>
int launch_norm_forward(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st) {
#define ROF_NORM_LAUNCH(LPR, WAVES, K)                                                                                          \
    if (s.lpr == LPR && s.waves == WAVES && s.k == K) {                                                                         \
        hipLaunchKernelGGL((norm_fwd_kernel<TX, TY, LPR, WAVES, K>), dim3(blocks), dim3((RowMap<TX, LPR, WAVES, K>::THREADS)), 0, \
                           st, a);                                                                                              \
        HIP_TRY(hipGetLastError());                                                                                             \
        return ROF_OK;                                                                                                          \
    }
    ROF_NORM_STREAMED(ROF_NORM_LAUNCH)
    ROF_NORM_OTHERS(ROF_NORM_LAUNCH)
    if constexpr (sizeof(TX) == 4) {
        ROF_NORM_F32(ROF_NORM_LAUNCH)
    } else {
        ROF_NORM_BF16(ROF_NORM_LAUNCH)
    }
#undef ROF_NORM_LAUNCH
    return ROF_ERR_UNSUPPORTED;
}

template <typename TX, typename TY, bool RELU>
int launch_norm_backward(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st) {
#define ROF_NORM_LAUNCH_AS(LPR, WAVES, K, STREAM)                                                                               \
    if (s.lpr == LPR && s.waves == WAVES && s.k == K && s.stream == STREAM) {                                                   \
        hipLaunchKernelGGL((norm_bwd_kernel<TX, TY, LPR, WAVES, K, RELU, STREAM>), dim3(blocks),                                \
                           dim3((RowMap<TX, LPR, WAVES, K>::THREADS)), 0, st, a);                                               \
        HIP_TRY(hipGetLastError());                                                                                             \
        return ROF_OK;                                                                                                          \
    }
#define ROF_NORM_LAUNCH(LPR, WAVES, K) ROF_NORM_LAUNCH_AS(LPR, WAVES, K, false)
#define ROF_NORM_LAUNCH_STREAMED(LPR, WAVES, K) ROF_NORM_LAUNCH_AS(LPR, WAVES, K, true)
    ROF_NORM_STREAMED(ROF_NORM_LAUNCH)
    ROF_NORM_STREAMED(ROF_NORM_LAUNCH_STREAMED)
    ROF_NORM_OTHERS(ROF_NORM_LAUNCH)
    if constexpr (sizeof(TX) == 4) {
        ROF_NORM_F32(ROF_NORM_LAUNCH)
    } else {
        ROF_NORM_BF16(ROF_NORM_LAUNCH)
    }
#undef ROF_NORM_LAUNCH_STREAMED
#undef ROF_NORM_LAUNCH
#undef ROF_NORM_LAUNCH_AS
    return ROF_ERR_UNSUPPORTED;
}

}  // namespace rofn

#endif
