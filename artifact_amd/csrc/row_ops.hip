// Operators on the feature rows between two graph convolutions: layer norm (forward, backward; kernels in norm_rows.h),
// dropout whose mask is computed and never stored, and the generator state the dropout reads.  C ABI in include/rof.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "rof.h"
#include "rof_internal.h"
#include "row_ops.h"

namespace {

using namespace rofn;

// Workgroups of the backward launch at most: each leaves a row of 2 f partial sums for the parameters' gradients.  From
// kManyRounds rounds of work on it is tiles of four rounds, else workgroups that stay; all of these: see norm_blocks.
constexpr int kBackwardBlocks = 1280, kBackwardTiles = 16384;
constexpr int64_t kPairedRounds = 20000, kFullRounds = 30000, kManyRounds = 100000;
constexpr int kTiledColumns = 512;   // rows of more columns are more than 64 vectors in either type
constexpr int kParamsChunks = 128;   // rows that the first of two passes leaves of so many partial ones
// An output of this size is beyond what the 256 MB Infinity Cache keeps beside its inputs until it is read again.
constexpr int64_t kStreamOutBytes = 128 << 20;
// A launch holds fewer than 2^32 threads.
constexpr int64_t kMostBlocks = 1 << 22;

struct DropoutArgs {
    const void *x;
    void *out;
    int64_t ldx, ldo;
    int64_t n;
    int64_t tiles;
    int32_t f;
    int32_t vecs;            // vectors of 16 bytes per row
    int32_t rows, parts;     // a tile is `rows` whole rows (parts = 1) or one of the `parts` parts of a row
    uint32_t magic;          // floor(2^32 / vecs) + 1 (0: a row is one vector)
    uint32_t threshold;
    float scale;
    const int64_t *state;
    int64_t call;
};

// A workgroup's tile is 1024 vectors (four per lane, loaded together) of whole rows next to each other, or a part of one long
// row.  Bounded by memory: half of its operations are the generator's (a call per vector; two float32 vectors make the same
// call, which is cheaper than eight columns per lane, whose loads would be 32 bytes apart).  Tiles rather than workgroups that
// stay and step through the matrix: 2^22 x 256 bfloat16 695 us a pass, 6.2 TB/s, against 900, 2.4 M x 100 float32 318, 6.0,
// against 450 (alone on the card; 765 and 330 under a profiler).  16384 x 32 float32: 4 us, a launch.
constexpr int kTileVecs = 1024;

template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    constexpr int V = 16 / (int)sizeof(T), U = kTileVecs / 256;
    const Drop d(a);
    const uint32_t groups = ((uint32_t)a.f + 7) / 8;
    const int tail = a.f % V;
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int64_t row0 = a.parts > 1 ? tile / a.parts : tile * a.rows;
        const uint32_t vec0 = a.parts > 1 ? (uint32_t)(tile - row0 * a.parts) * kTileVecs : 0;
        const uint32_t count = a.parts > 1 ? std::min((uint32_t)a.vecs - vec0, (uint32_t)kTileVecs)
                                           : (uint32_t)std::min<int64_t>(a.n - row0, a.rows) * (uint32_t)a.vecs;
        const T *const src = (const T *)a.x + row0 * a.ldx;
        T *const dst = (T *)a.out + row0 * a.ldo;
        const uint64_t group0 = (uint64_t)row0 * groups;
        Packed<T, V> p[U];
        uint32_t row[U], col[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = std::min(u * 256 + threadIdx.x, count - 1);   // behind the tile: its last vector once more, not stored
            row[u] = a.parts > 1 ? 0 : a.magic ? __umulhi(i, a.magic) : i;   // i / vecs: exact, since i and vecs are at most 1024
            col[u] = (vec0 + i - row[u] * (uint32_t)a.vecs) * V;
            const T *const at = src + (uint64_t)row[u] * (uint64_t)a.ldx;
            // the last vector of a row that is no multiple of V: read from the row's end and shifted into place
            if (a.f < V)
                p[u].load_few(at, a.f);
            else
                p[u].template load<STREAM>(at + std::min(col[u], (uint32_t)(a.f - V)));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool cut = col[u] + V > (uint32_t)a.f;
            if (tail && a.f >= V) p[u].shift(cut ? V - tail : 0);
            float v[V];
            p[u].unpack(v);
            if (a.threshold) {
                bool keep[V];
                drop_kept(d, group0 + (uint64_t)row[u] * groups, col[u], keep);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = keep[e] ? v[e] * a.scale : 0.f;
            }
            p[u].pack(v);
            if (u * 256 + threadIdx.x < count) {
                T *const at = dst + (uint64_t)row[u] * (uint64_t)a.ldo + col[u];
                if (cut)
                    p[u].store_part(at, tail);
                else
                    p[u].template store<STREAM>(at);
            }
        }
    }
}

__global__ void dropout_state_next_kernel(int64_t *state, int64_t calls, int64_t *used) {
    const int64_t seed = state[0], offset = state[1];
    used[0] = seed;
    used[1] = offset;
    state[1] = (int64_t)((uint64_t)offset + (uint64_t)calls);
}

// Sums of the partial rows, column by column in a fixed order: 16 columns x 64 slices of the rows per workgroup (the
// columns are few, so narrow workgroups are what makes enough of them).  3 us (256 rows of 32) to 9 us (512 rows of 8198);
// 1024 rows of 128 take 5 us with eight loads under way per lane, 7 with the compiler's choice.  In 64 bits, which costs 0 to
// 0.3 us and leaves of the gradients' error what the workgroups' own sums have (16384 x 16 float32, the bias's: 5.8e-8 of its
// norm, in 32 bits 1.9e-7).
__global__ __launch_bounds__(1024) void norm_params_kernel(const float *__restrict__ partial, int blocks, int f,
                                                            float *__restrict__ dweight, float *__restrict__ dbias) {
    __shared__ double red[64][16];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int c = blockIdx.x * 16 + tx;
    double s = 0.0;
    if (c < 2 * f) {
#pragma unroll 8
        for (int b = ty; b < blocks; b += 64) s += partial[(int64_t)b * 2 * f + c];
    }
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < 2 * f) {
        s = 0.0;
#pragma unroll
        for (int i = 0; i < 64; ++i) s += red[i][tx];
        if (c < f) {
            if (dweight) dweight[c] = (float)s;
        } else if (dbias) {
            dbias[c - f] = (float)s;
        }
    }
}

// Thousands of partial rows are first added up in kParamsChunks chunks, 64 columns of a chunk per workgroup (4096 rows of
// 512 floats: 5 us, and 5 us for the other kernel behind it; that one alone would have them in 32 workgroups).
__global__ __launch_bounds__(256) void norm_params_chunk_kernel(const float *__restrict__ partial, int blocks, int f,
                                                                 float *__restrict__ out) {
    __shared__ double red[4][64];
    const int tx = threadIdx.x % 64, ty = threadIdx.x / 64;
    const int c = blockIdx.x * 64 + tx, per = (blocks + kParamsChunks - 1) / kParamsChunks;
    const int first = blockIdx.y * per, last = std::min(blocks, first + per);
    double s = 0.0;
    if (c < 2 * f) {
#pragma unroll 8
        for (int b = first + ty; b < last; b += 4) s += partial[(int64_t)b * 2 * f + c];
    }
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < 2 * f) out[(int64_t)blockIdx.y * 2 * f + c] = (float)((red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]));
}

bool known_type(int t) { return t == ROF_F32 || t == ROF_BF16; }
int size_of(int t) { return t == ROF_F32 ? 4 : 2; }
bool aligned(const void *p, int size) { return ((uintptr_t)p) % (uintptr_t)size == 0; }

// The threshold of a rate, or -1: the rate is taken to the nearest multiple of 2^-16.
int drop_threshold(const rof_dropout_opts *d) {
    if (!(d->p >= 0.0 && d->p <= 1.0)) return -1;
    const int t = (int)(d->p * 65536.0 + 0.5);
    if (t > 0 && (!d->state || !aligned(d->state, 8))) return -1;
    return t;
}
float drop_scale(int threshold) { return threshold < 65536 ? (float)(65536.0 / (65536 - threshold)) : 0.f; }

// The variant for f columns.  A row of up to 64 vectors of 16 bytes is one vector in each lane of the smallest lane group
// that holds it: few registers, and the rows of a wavefront are one contiguous piece.  Measured (us, forward / backward, each
// with the launch size that suits it best):
//   2^20 x 64 bfloat16, 8 vectors: 8 lanes 40 / 70, 4 lanes with two vectors 39 / 75, 16 lanes half empty 50 / 96;
//   2^22 x 256 bfloat16, 32 vectors, with ReLU and dropout: 32 lanes 738 / 1111, 16 with two 739 / 1141;
//   2^18 x 256 float32, 64 vectors: 64 lanes 92 / 134, 32 lanes with two vectors 92 / 131.
// A group of 16 or more lanes of which that would leave a quarter idle is half as many lanes with two vectors (float32) or a
// quarter with three (bfloat16, whose arithmetic per byte is twice as much); with ReLU and dropout:
//   667 000 x 150 float32, 38 vectors: 32 lanes with two 147 / 234, 64 lanes 173 / 275, 16 with three 146 / 233;
//   667 000 x 300 bfloat16, 38 vectors: 16 lanes with three 153 / 245, 64 lanes 209 / 348, 32 with two 180 / 322.
// Above that two or three vectors per lane and as few wavefronts as that takes, because every wavefront more waits for the
// others twice per row, and as few idle lanes; bfloat16:
//   385 000 x 520, 65 vectors, with ReLU and dropout: 32 lanes with three 153 / 246, 64 with two 188 / 340;
//   39 000 x 2048, 256 vectors: two wavefronts with two vectors 57 / 83, one with four 54 / 93, four with one 56 / 83;
//   20011 x 4099, 513 vectors: three with three 62 / 112, four with three 67 / 117, eight with two 89 / 159;
//   9765 x 8192, 1024 vectors: eight with two 54 / 86, four with four 55 / 98.
NormShape norm_shape(int f, int x_dtype) {
    // In every entry the vectors of a lane but its last are whole, because the entry before it ends at (k - 1) lpr waves or later.
    struct Shape { int most, lpr, waves, k; };
    static const Shape kF32[] = {{1, 1, 1, 1},   {2, 2, 1, 1},   {4, 4, 1, 1},   {8, 8, 1, 1},   {11, 8, 1, 2}, {16, 16, 1, 1},
                                 {23, 16, 1, 2}, {32, 32, 1, 1}, {47, 32, 1, 2}, {64, 64, 1, 1}};
    static const Shape kBf16[] = {{1, 1, 1, 1},  {2, 2, 1, 1},   {4, 4, 1, 1},   {8, 8, 1, 1},  {12, 4, 1, 3}, {16, 16, 1, 1},
                                  {24, 8, 1, 3}, {32, 32, 1, 1}, {48, 16, 1, 3}, {64, 64, 1, 1}};
    static const Shape kWide[] = {{96, 32, 1, 3},  {128, 64, 1, 2}, {192, 64, 1, 3}, {256, 64, 2, 2},  {384, 64, 3, 2}, {512, 64, 4, 2},
                                  {576, 64, 3, 3}, {768, 64, 4, 3}, {1024, 64, 8, 2}, {1536, 64, 8, 3}, {2048, 64, 8, 4}};
    const int vecs = (f * size_of(x_dtype) + 15) / 16;
    const Shape *c = vecs > 64 ? kWide : x_dtype == ROF_F32 ? kF32 : kBf16;
    while (vecs > c->most) ++c;   // ends: a row is at most 2048 vectors
    return {c->lpr, c->waves, c->k, false};
}

// Up to 64 vectors, in whichever of the shapes.
bool is_lean(const NormShape &s) { return s.waves * s.lpr * s.k <= 64; }
int64_t rounds_of(const NormShape &s, int64_t n) { return (n + s.rows() - 1) / s.rows(); }
// Whether the backward launch is tiles, see norm_blocks.
bool is_tiled(const NormShape &s, int64_t n) { return is_lean(s) && rounds_of(s, n) >= kManyRounds; }

// How many workgroups, and which rounds each takes.
// Forward: a workgroup per four adjacent rounds where that makes thousands of them (2^22 x 256 bfloat16: 743 us against 862
// with 2048 workgroups that stay and step through the matrix together; 10^6 x 100 float32 142 / 155), else as many as stay:
// 2048, or half as many where the lanes hold several vectors.
// Backward: each workgroup leaves a row of partial sums.  With many rounds it is tiles of four adjacent ones, handed out as
// others end: up to 16384 for float32 (10^6 x 200 424 us; 4096 tiles 471, 1280 workgroups that stay 478; 2.4 M x 100 512 / 564 /
// 570), up to 4096 for bfloat16, whose workgroups are fewer on a CU (1.6 M x 300 602, 16384 tiles 653, 1024 that stay 602; 2.4 M x
// 47 171 / 184 / 170; 2^22 x 256 1132 / 1119 / 1207), and more launches and traffic for their sums.  kManyRounds is one number for four crossings (geometric
// means over 15 widths and types): 80000 rounds for two float32 vectors a lane, 130000 for one, 140000 for three bfloat16 ones,
// and between 250000 and 500000 for one, where tiles take 1.06 of the time at 100000 and 0.93 at 524288.  With fewer rounds
// workgroups stay, as many as fit: four on a CU (1024), two (512) where a lane holds several bfloat16 vectors, whose registers
// leave room for no more.  Rows of up to 64 vectors, a dozen widths with and without ReLU and dropout, geometric means of the
// times against one round at a time with 1024 workgroups, by the number of rounds:
//                                          4000  16000  20000  24000  28000  32768  50000  65536  80000  99000
//   two adjacent rounds    float32         1.00   1.01   1.00   0.99   0.99   1.00   0.99   0.99   0.99   0.99
//                          bfloat16        1.00   1.01   1.00   0.98   1.00   0.98   0.98   0.98   0.98   0.98
//   four                   float32         1.08   1.02   1.02   1.01   1.02   1.01   1.00   0.99   0.98   0.98
//                          bfloat16        1.07   1.02   1.01   1.01   1.04   0.99   0.99   0.98   0.97   0.97
//   two, 1280 workgroups   float32         1.05   1.04   1.03   1.01   1.01   0.98   0.98   0.97   0.98   0.98
//     two vectors a lane   float32         1.13   1.13   1.16   1.19   1.12   1.11   1.12   1.10   1.10   1.10
//                          bfloat16        1.09   1.12   1.08   1.14   1.14   1.09   1.12   1.09   1.10   1.10
//   two, 512 workgroups    float32         1.01   1.09   1.09   1.15   1.20   1.26   1.28   1.27   1.26   1.26
//     three vectors a lane bfloat16        0.86   0.96   0.95   0.95   0.96   0.96   0.97   0.97   0.97   0.98
// So two rounds from kPairedRounds on, and five workgroups on a CU for one float32 vector from kFullRounds on.  Wide rows: two
// rounds (20011 x 4099 bfloat16 with four wavefronts: 106 us against 117 one at a time; forward with three 62 / 71) and two
// workgroups on a CU (65 to 192 vectors, which are one wavefront's or less, nine widths and pairs of types at 8000 to 120000
// rounds: 0.84 to 1.01 of the time that 1024 take), but four of those of two wavefronts (with ReLU and dropout 512 take 1.3 to
// 1.75 times as long).
int norm_blocks(NormArgs &a, const NormShape &s, int x_dtype, bool backward) {
    const int64_t rows = s.rows(), rounds = rounds_of(s, a.n);
    const bool lean = is_lean(s), f32 = x_dtype == ROF_F32;
    int64_t most;
    if (!backward && rounds / 4 >= 4096 && rounds / 4 < kMostBlocks) {
        a.inner = 4;
        most = kMostBlocks;
    } else if (!backward) {
        a.inner = lean || rounds < 2048 ? 1 : 2;
        most = lean ? 2048 : 1024;
    } else if (lean) {
        const bool tiled = is_tiled(s, a.n);
        a.inner = tiled ? 4 : rounds >= kPairedRounds ? 2 : 1;
        if (tiled)
            most = f32 ? kBackwardTiles : kBackwardTiles / 4;
        else if (f32)
            most = s.k == 1 && rounds >= kFullRounds ? kBackwardBlocks : 1024;
        else
            most = s.k == 1 ? 1024 : 512;
    } else {
        a.inner = rounds < 2048 ? 1 : 2;
        most = s.waves == 2 ? 1024 : 512;
    }
    const int blocks = (int)std::min<int64_t>((rounds + a.inner - 1) / a.inner, most);
    a.jump = ((int64_t)blocks * a.inner - (a.inner - 1)) * rows;
    return blocks;
}

// Streaming accesses in the backward launch: where its result is larger than the caches keep until its consumer runs, its
// inputs are read for the last time as well, and whole rows are whole cache lines (2^18 x 256 float32: 146 us against 154,
// 2^20 x 64 bfloat16 66 / 74; rows of 47 columns, whose lines two wavefronts share, 288 / 258).
bool norm_streams(const NormArgs &a, const NormShape &s, int x_dtype, int y_dtype) {
    const int sx = size_of(x_dtype), sy = size_of(y_dtype);
    if (a.n * a.f * sx < kStreamOutBytes || s.k > 2 || s.lpr < 8 || (s.k > 1 && s.lpr < 64)) return false;
    return aligned(a.x, 16) && aligned(a.dout, 16) && aligned(a.out, 16) && a.ldx * sx % 16 == 0 && a.ldd * sy % 16 == 0 &&
           a.ldo * sx % 16 == 0 && (int64_t)a.f * sx % 16 == 0;
}

int launch_norm(NormArgs &a, int x_dtype, int y_dtype, hipStream_t st) {
    const NormShape s = norm_shape(a.f, x_dtype);
    const int blocks = norm_blocks(a, s, x_dtype, false);
    if (x_dtype == ROF_F32) return y_dtype == ROF_F32 ? norm_fwd_f32_f32(a, s, blocks, st) : norm_fwd_f32_bf16(a, s, blocks, st);
    return y_dtype == ROF_F32 ? norm_fwd_bf16_f32(a, s, blocks, st) : norm_fwd_bf16_bf16(a, s, blocks, st);
}

int launch_norm_backward(NormArgs &a, int x_dtype, int y_dtype, hipStream_t st, int *blocks) {
    NormShape s = norm_shape(a.f, x_dtype);
    s.stream = norm_streams(a, s, x_dtype, y_dtype);
    const int b = *blocks = norm_blocks(a, s, x_dtype, true);
    if (x_dtype == ROF_F32) {
        if (y_dtype == ROF_F32) return a.relu ? norm_bwd_relu_f32_f32(a, s, b, st) : norm_bwd_f32_f32(a, s, b, st);
        return a.relu ? norm_bwd_relu_f32_bf16(a, s, b, st) : norm_bwd_f32_bf16(a, s, b, st);
    }
    if (y_dtype == ROF_F32) return a.relu ? norm_bwd_relu_bf16_f32(a, s, b, st) : norm_bwd_bf16_f32(a, s, b, st);
    return a.relu ? norm_bwd_relu_bf16_bf16(a, s, b, st) : norm_bwd_bf16_bf16(a, s, b, st);
}

// the arguments that the two directions share
int norm_args(NormArgs &a, const void *x, int x_dtype, int64_t ldx, int64_t n, int f, const float *weight, const float *bias,
              double eps, int relu, const rof_dropout_opts *dropout, int y_dtype) {
    if (n < 0 || f < 1 || ldx < f || (n && !x) || !(eps >= 0.0 && eps <= 1e30)) return ROF_ERR_ARG;
    if (!known_type(x_dtype) || !known_type(y_dtype) || f > ROF_LAYER_NORM_MAX_ROW_BYTES / size_of(x_dtype))
        return ROF_ERR_UNSUPPORTED;
    if (!aligned(x, size_of(x_dtype)) || !aligned(weight, 4) || !aligned(bias, 4)) return ROF_ERR_ARG;
    a = NormArgs();
    a.x = x;
    a.ldx = ldx;
    a.n = n;
    a.f = f;
    a.weight = weight;
    a.bias = bias;
    a.eps = eps;
    a.relu = relu != 0;
    a.scale = 1.f;
    if (dropout) {
        const int t = drop_threshold(dropout);
        if (t < 0) return ROF_ERR_ARG;
        a.drop = t > 0;
        a.threshold = (uint32_t)t;
        a.scale = drop_scale(t);
        a.state = t > 0 ? dropout->state : nullptr;
        a.call = dropout->call;
    }
    return ROF_OK;
}

}  // namespace

extern "C" {

int rof_dropout_state_next(int64_t *state, int64_t calls, int64_t *used, void *stream) {
    if (!state || !used || calls < 0 || !aligned(state, 8) || !aligned(used, 8)) return ROF_ERR_ARG;
    if ((uintptr_t)used < (uintptr_t)state + 16 && (uintptr_t)state < (uintptr_t)used + 16) return ROF_ERR_ARG;   // overlapping
    hipLaunchKernelGGL(dropout_state_next_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, state, calls, used);
    HIP_TRY(hipGetLastError());
    return ROF_OK;
}

int rof_dropout(const void *x, int dtype, int64_t ldx, int64_t n, int f, void *out, int64_t ldo,
                const rof_dropout_opts *dropout, void *stream_) {
    if (!dropout || n < 0 || f < 1 || ldx < f || ldo < f || (n && (!x || !out))) return ROF_ERR_ARG;
    if (!known_type(dtype)) return ROF_ERR_UNSUPPORTED;
    const int t = drop_threshold(dropout);
    if (t < 0 || !aligned(x, size_of(dtype)) || !aligned(out, size_of(dtype))) return ROF_ERR_ARG;
    if (n == 0) return ROF_OK;
    DropoutArgs a;
    a.x = x;
    a.out = out;
    a.ldx = ldx;
    a.ldo = ldo;
    a.n = n;
    a.f = f;
    const int per = 16 / size_of(dtype);
    a.vecs = f / per + (f % per != 0);
    a.rows = std::max(1, kTileVecs / a.vecs);
    a.parts = (a.vecs + kTileVecs - 1) / kTileVecs;
    a.tiles = a.parts > 1 ? n * a.parts : (n + a.rows - 1) / a.rows;
    a.magic = a.vecs > 1 ? (uint32_t)(((uint64_t)1 << 32) / a.vecs) + 1 : 0;
    a.threshold = (uint32_t)t;
    a.scale = drop_scale(t);
    a.state = t > 0 ? dropout->state : nullptr;
    a.call = dropout->call;
    const bool stream = n * f * size_of(dtype) >= kStreamOutBytes && aligned(x, 16) && aligned(out, 16) && f % per == 0 &&
                        ldx % per == 0 && ldo % per == 0;
    const dim3 grid((unsigned)std::min(a.tiles, kMostBlocks));
    hipStream_t st = (hipStream_t)stream_;
    if (dtype == ROF_F32 && stream)
        hipLaunchKernelGGL((dropout_kernel<float, true>), grid, dim3(256), 0, st, a);
    else if (dtype == ROF_F32)
        hipLaunchKernelGGL((dropout_kernel<float, false>), grid, dim3(256), 0, st, a);
    else if (stream)
        hipLaunchKernelGGL((dropout_kernel<bf16_t, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((dropout_kernel<bf16_t, false>), grid, dim3(256), 0, st, a);
    HIP_TRY(hipGetLastError());
    return ROF_OK;
}

int rof_layer_norm(const void *x, int x_dtype, int64_t ldx, int64_t n, int f, const float *weight, const float *bias, double eps,
                   int relu, const rof_dropout_opts *dropout, void *out, int out_dtype, int64_t ldo, void *stream) {
    NormArgs a;
    const int rc = norm_args(a, x, x_dtype, ldx, n, f, weight, bias, eps, relu, dropout, out_dtype);
    if (rc) return rc;
    if (ldo < f || (n && !out) || !aligned(out, size_of(out_dtype))) return ROF_ERR_ARG;
    if (n == 0) return ROF_OK;
    a.out = out;
    a.ldo = ldo;
    return launch_norm(a, x_dtype, out_dtype, (hipStream_t)stream);
}

size_t rof_layer_norm_backward_workspace_bytes(int64_t n, int f) {
    if (n <= 0 || f <= 0) return 0;
    // for rows of either type
    const bool tiled = f <= kTiledColumns && (is_tiled(norm_shape(f, ROF_F32), n) || is_tiled(norm_shape(f, ROF_BF16), n));
    const int64_t rows = tiled ? kBackwardTiles + kParamsChunks : std::min<int64_t>(n, kBackwardBlocks);
    return (size_t)rows * 2 * (size_t)f * sizeof(float);
}

int rof_layer_norm_backward(const void *dout, int dout_dtype, int64_t ldd, const void *x, int x_dtype, int64_t ldx, int64_t n,
                            int f, const float *weight, const float *bias, double eps, int relu, const rof_dropout_opts *dropout,
                            void *dx, int64_t lddx, float *dweight, float *dbias, void *workspace, size_t workspace_bytes,
                            void *stream) {
    NormArgs a;
    const int rc = norm_args(a, x, x_dtype, ldx, n, f, weight, bias, eps, relu, dropout, dout_dtype);
    if (rc) return rc;
    if (ldd < f || (n && !dout) || !aligned(dout, size_of(dout_dtype)) || (dx && (lddx < f || !aligned(dx, size_of(x_dtype)))) ||
        !aligned(dweight, 4) || !aligned(dbias, 4))
        return ROF_ERR_ARG;
    const bool params = dweight || dbias;
    if (params && n && (!workspace || !aligned(workspace, 16) || workspace_bytes < rof_layer_norm_backward_workspace_bytes(n, f)))
        return ROF_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    int blocks = 0;
    if (n && (params || dx)) {
        a.dout = dout;
        a.ldd = ldd;
        a.out = dx;
        a.ldo = lddx;
        a.partial = params ? (float *)workspace : nullptr;
        const int status = launch_norm_backward(a, x_dtype, dout_dtype, st, &blocks);
        if (status) return status;
    }
    if (params) {
        const float *partial = (const float *)workspace;
        if (blocks > kBackwardBlocks) {
            float *chunks = (float *)workspace + (int64_t)kBackwardTiles * 2 * f;
            hipLaunchKernelGGL(norm_params_chunk_kernel, dim3((2 * f + 63) / 64, kParamsChunks), dim3(256), 0, st, partial, blocks, f,
                               chunks);
            HIP_TRY(hipGetLastError());
            partial = chunks;
            blocks = kParamsChunks;
        }
        hipLaunchKernelGGL(norm_params_kernel, dim3((2 * f + 15) / 16), dim3(1024), 0, st, partial, blocks, f, dweight, dbias);
        HIP_TRY(hipGetLastError());
    }
    return ROF_OK;
}

}  // extern "C"
