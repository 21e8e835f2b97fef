// What stands between two blocks, in one pass over the rows: the RMS norm after a block, its gate and scale, the sum
// with the residual, and the RMS norm before the next block.
//
//   p = y * inv1 * w_post            inv1 = 1 / sqrt(mean(y^2) + eps)      (without w_post: p = y)
//   h = residual + scale * g * p     g: one per channel, one per token, or 1
//   n = h * inv2 * w_pre             inv2 = 1 / sqrt(mean(h^2) + eps)      (without w_pre: no n)
//
// and the gradient.  With u = y * inv1, v = h * inv2, t = dn * w_pre and q = scale * g * p:
//   dH = dh + inv2 * (t - v * mean(t v));  d_residual = dH;  dp = scale * g * dH
//   d_y = inv1 * (dp * w_post - u * mean(dp w_post u));  d_w_post = sum dp u;  d_w_pre = sum dn v;  d_g = sum scale p dH
// The two means need three sums that do not wait for each other -- sum(t v), sum((dh + inv2 t) q), sum(v q) -- because
// sum(dH q) = sum((dh + inv2 t) q) - inv2 * mean(t v) * sum(v q), so a row costs one reduction.
//
// Without a gradient of n (or without w_pre) t is not there: dH = dh, and neither h nor v is made.
//
// All arithmetic is fp32; every output is rounded once.  n comes from the unrounded h, and the gradient recomputes h
// from y and the residual, so no stored rounding enters it.  With a post norm or a gate y is needed anyway and the
// residual is read in the place of h, the same bytes; with neither, y and the residual are read where h alone would do.
#include "common.hpp"

namespace terrace {

constexpr int kNormThreads = 1024, kNormWaves = kNormThreads / kWave;

struct NormArgs {
    const void *y, *residual, *w_post, *gate, *w_pre;        // any but residual may be NULL
    int post_dtype, gate_dtype, pre_dtype, gate_kind;
    float scale, eps;
    int64_t T, H;
    int tpr;                                                 // threads per row: whole waves
    int groups;                                              // rows a workgroup works on at a time
};

// A lane's share of a row: E elements as E / 8 pieces of 8 neighbours, piece i at (lane + i * tpr) * 8.  The bits are kept
// as loaded until they are used, which for 16-bit rows halves the registers of a row that is fetched ahead.  ALIGNED:
// rows are multiples of 8 elements on 16-byte boundaries; otherwise a piece is loaded and stored as a vector with the
// alignment of its elements, and the last piece of a row element by element.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_word __attribute__((ext_vector_type(4), aligned(4)));

template <int DT, bool ALIGNED>
__device__ __forceinline__ void load_piece(const uint8_t *row, int c, int64_t H, uint32_t *w) {
    constexpr int kVecs = DT == TERRACE_F32 ? 2 : 1, kBytes = DT == TERRACE_F32 ? 4 : 2;
#pragma unroll
    for (int j = 0; j < 4 * kVecs; ++j) w[j] = 0;
    if (ALIGNED ? c < H : c + 8 <= H) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const uint8_t *p = row + c * kBytes + v * 16;
            u32x4 x;
            if constexpr (ALIGNED) x = ld_stream((const u32x4 *)p);
            else if constexpr (DT == TERRACE_F32) x = *(const u32x4_word *)p;
            else x = *(const u32x4_any *)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * v + j] = x[j];
        }
    } else if (!ALIGNED && c < H) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (c + j >= H) continue;
            if constexpr (DT == TERRACE_F32) w[j] = ((const uint32_t *)row)[c + j];
            else w[j / 2] |= (uint32_t)((const uint16_t *)row)[c + j] << (j & 1 ? 16 : 0);
        }
    }
}

template <int DT, bool ALIGNED, int E>
struct Share {
    static constexpr int kPiece = DT == TERRACE_F32 ? 8 : 4;
    uint32_t w[E / 8 * kPiece];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < E / 8 * kPiece; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const void *rows, int64_t row, int64_t H, int at, int tpr) {
#pragma unroll
        for (int i = 0; i < E / 8; ++i)
            load_piece<DT, ALIGNED>((const uint8_t *)rows + row * H * (DT == TERRACE_F32 ? 4 : 2), (at + i * tpr) * 8, H,
                                    w + i * kPiece);
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (DT == TERRACE_F32) {
            return __uint_as_float(w[e]);
        } else {
            const uint32_t b = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
            if constexpr (DT == TERRACE_BF16) return bf16_bits_to_f32(b);
            else return __half2float(__ushort_as_half((unsigned short)b));
        }
    }
};

template <int DT, bool ALIGNED, int E>
__device__ __forceinline__ void store_share(void *rows, int64_t row, int64_t H, int at, int tpr, const float *f) {
    uint8_t *base = (uint8_t *)rows + row * H * (DT == TERRACE_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        const int c = (at + i * tpr) * 8;
        if constexpr (ALIGNED) {
            if (c < H) store_floats<DT, 8>(base, c, f + i * 8);
        } else if (c + 8 <= H) {
            if constexpr (DT == TERRACE_F32) {
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    u32x4 x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = __float_as_uint(f[i * 8 + 4 * v + j]);
                    *(u32x4_word *)(base + c * 4 + v * 16) = x;
                }
            } else {
                u32x4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = to_bits16x2<DT>(f[i * 8 + 2 * j], f[i * 8 + 2 * j + 1]);
                *(u32x4_any *)(base + c * 2) = x;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (c + j < H) store_floats<DT, 1>(base, c + j, f + i * 8 + j);
            }
        }
    }
}

// A vector over the channels (a weight, a gate) in the same shares; absent: `fill`.
template <bool ALIGNED, int E>
__device__ __forceinline__ void load_channels(const void *v, int dtype, int64_t H, int at, int tpr, float fill, float *f) {
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        const int c = (at + i * tpr) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i * 8 + j] = fill;
        if (!v) continue;
        if constexpr (ALIGNED) {
            if (c >= H) continue;
            if (dtype == TERRACE_F32) load_floats<TERRACE_F32, 8>(v, c, f + i * 8);
            else if (dtype == TERRACE_BF16) load_floats<TERRACE_BF16, 8>(v, c, f + i * 8);
            else load_floats<TERRACE_F16, 8>(v, c, f + i * 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (c + j >= H) continue;
                if (dtype == TERRACE_F32) load_floats<TERRACE_F32, 1>(v, c + j, f + i * 8 + j);
                else if (dtype == TERRACE_BF16) load_floats<TERRACE_BF16, 1>(v, c + j, f + i * 8 + j);
                else load_floats<TERRACE_F16, 1>(v, c + j, f + i * 8 + j);
            }
        }
    }
}

__device__ __forceinline__ float load_scalar(const void *v, int dtype, int64_t i) {
    float f;
    if (dtype == TERRACE_F32) load_floats<TERRACE_F32, 1>(v, i, &f);
    else if (dtype == TERRACE_BF16) load_floats<TERRACE_BF16, 1>(v, i, &f);
    else load_floats<TERRACE_F16, 1>(v, i, &f);
    return f;
}

// Sum of M values over the tpr threads of a row, in every thread; called by all threads of the workgroup.  `part` holds
// M floats per wave; two buffers used in turn need no barrier between one sum and the next.
template <int M>
__device__ __forceinline__ void row_sum(float *v, float *part, int tpr) {
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] = wave_sum(v[m]);
    if (tpr == kWave) return;
    const int w = wave_in_block(), n = tpr / kWave, w0 = w / n * n, lane = lane_id() & 15;       // n <= 16 waves
    if (lane_id() == 0) {
#pragma unroll
        for (int m = 0; m < M; ++m) part[m * kNormWaves + w] = v[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] = row16_sum(lane < n ? part[m * kNormWaves + w0 + lane] : 0.0f);
}

// A workgroup walks the rows (blockIdx.x + i * gridDim.x) * groups + group, with rows in flight while its waves meet: the next
// one, fetched at the start of a row (AHEAD 1), or the next two, a row's registers taking the row after the next as soon
// as h is made of them (AHEAD 2).  16384 rows of 7168 bf16, 940 MB, 64 rows a workgroup: 162-170 us with two (5.8 TB/s),
// 173-183 us with one, 287 us with none and a workgroup a row.  Two ahead are taken over more than 2048 groups of rows where a
// row's bits are few, that is 16-bit rows beside a 16-bit residual, and not both unaligned and 16 elements a lane
// (norm_two_ahead); two / one ahead, us:
//   taken      16384 x 12288 bf16 290 / 304, x 16384 406 / 415, x 7167 361 / 383; 4096 x 7168 47.4 / 47.9, x 16384 101 / 100
//   not taken  16384 x 7168 beside f32 283 / 268, f32 388 / 362; x 16384 beside f32 667 / 633, f32 986 / 849; x 12289 bf16 499 / 448
// (the f32 and the unaligned wide forms with two ahead spill 14 to 83 registers a lane).  Over fewer groups one is as fast
// or faster: 4096 x 1024 bf16 10.9 / 9.9, f32 19 / 17.
constexpr bool norm_two_ahead(int r_dtype, bool aligned, int per) { return r_dtype != TERRACE_F32 && (aligned || per == 8); }

template <int TY, int TR, bool ALIGNED, int E, int AHEAD>
__global__ __launch_bounds__(kNormThreads) void block_norm_kernel(NormArgs a, void *__restrict__ h_out,
                                                                  void *__restrict__ n_out, float *__restrict__ stats) {
    __shared__ float part[2][kNormWaves];
    const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.x / a.tpr);          // whole waves per row
    const int at = (int)threadIdx.x - group * a.tpr;
    const float inv_h = 1.0f / (float)a.H;
    const int64_t stride = (int64_t)gridDim.x * a.groups;
    struct Row {
        Share<TY, ALIGNED, E> y;
        Share<TR, ALIGNED, E> r;
        float token;
    };
    auto fetch = [&](int64_t row, Row &x) {
        x.y.clear(), x.r.clear();
        x.token = 1.0f;
        if (row >= a.T) return;
        if (a.y) x.y.load(a.y, row, a.H, at, a.tpr);
        x.r.load(a.residual, row, a.H, at, a.tpr);
        if (a.gate_kind == TERRACE_GATE_TOKEN) x.token = load_scalar(a.gate, a.gate_dtype, row);
    };
    const int64_t first = (int64_t)blockIdx.x * a.groups;
    Row ring[2];
    fetch(first + group, ring[0]);
    float w[E], wn[E];                                       // scale, norm weight and gate per channel; the norm before
    load_channels<ALIGNED, E>(a.w_post, a.post_dtype, a.H, at, a.tpr, 1.0f, w);
    {
        float g[E];
        load_channels<ALIGNED, E>(a.gate_kind == TERRACE_GATE_CHANNEL ? a.gate : nullptr, a.gate_dtype, a.H, at, a.tpr, 1.0f, g);
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] *= a.scale * g[e];
    }
    load_channels<ALIGNED, E>(a.w_pre, a.pre_dtype, a.H, at, a.tpr, 0.0f, wn);
    if constexpr (AHEAD == 2) fetch(first + stride + group, ring[1]);                    // behind the vectors: loads return in order
    auto step = [&](int64_t base, Row &cur) {
        const int64_t row = base + group;
        const bool mine = row < a.T;
        if constexpr (AHEAD == 1) fetch(row + stride, ring[1]);
        float h[E], inv1 = 1.0f, inv2 = 1.0f;
        if (a.w_post) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = __fmaf_rn(cur.y.get(e), cur.y.get(e), s);
            row_sum<1>(&s, part[0], a.tpr);
            inv1 = 1.0f / sqrtf(__fmaf_rn(s, inv_h, a.eps));
        }
        const float factor = inv1 * cur.token;
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = a.y ? __fmaf_rn(w[e], cur.y.get(e) * factor, cur.r.get(e)) : cur.r.get(e);
        if constexpr (AHEAD == 2) fetch(row + 2 * stride, cur);          // its registers are free
        if (mine && h_out) store_share<TR, ALIGNED, E>(h_out, row, a.H, at, a.tpr, h);
        if (a.w_pre) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = __fmaf_rn(h[e], h[e], s);
            row_sum<1>(&s, part[1], a.tpr);
            inv2 = 1.0f / sqrtf(__fmaf_rn(s, inv_h, a.eps));
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = h[e] * inv2 * wn[e];
            if (mine) store_share<TY, ALIGNED, E>(n_out, row, a.H, at, a.tpr, h);
        }
        if (!a.w_post || !a.w_pre) __syncthreads();          // one sum a row: its buffer is used again at once
        if (mine && stats && at == 0) {
            stats[2 * row] = inv1;
            stats[2 * row + 1] = inv2;
        }
    };
    for (int64_t base = first; base < a.T; base += AHEAD * stride) {
        step(base, ring[0]);
        if constexpr (AHEAD == 2) {
            if (base + stride < a.T) step(base + stride, ring[1]);
        } else {
            ring[0] = ring[1];
        }
    }
}

// The gradient: 16384 rows of 7168 bf16, 1.41 GB, in 271-280 us, 5.0-5.2 TB/s.  By counters vector instructions fill
// 54 % of the cycles; the 14 waves of a row, alone on their CU, wait for each other once a row, which is likely the rest but
// was not measured apart.  512 workgroups took 385 us where 256 took 374-379.  Rows of 7167 take 618 us, 4096 rows of 1024 f32
// 31 us for 1001's 35: the unaligned and the f32 forms spill 6 to 26 registers a lane.
// A workgroup walks the rows blockIdx.x * groups + group + i * gridDim.x * groups.  The next row is fetched
// before the present one is reduced: the workgroup fills a CU, and without that nothing would be in flight while its
// waves meet.  The vectors over the channels wait in LDS.  The sums over the rows stay in registers over the walk, two of
// them, because d_w_post and the gradient of a gate per channel are both multiples of sum(dH u): each workgroup leaves one
// row partial[2][gridDim.x][H] of sum(factor dH u) and sum(dn v), and norm_reduce_kernel adds those up in order.
// WIDE (16 elements a lane): the sums are kept in the partial row itself, which the lane that owns the channel reads and
// writes row by row, the vectors are loaded again for every row, and no row is fetched ahead; 45 registers a lane spill, 231 to
// 245 with unaligned rows.  8192 rows of 12288 bf16 take 1141 us (1.1 TB/s of the rows' bytes), of 16384 bf16 1487, f32 1922, of
// 12289 bf16 2139: this form is right and no more.
//
// DN: there is a gradient of n.  Without one the residual is not read and nothing of h is formed, so an infinity or a NaN
// in it (or in y, without a post norm) reaches no sum that it is not a term of: 16384 rows of 7168 bf16 with a post norm, 940
// MB, 179 us (5.3 TB/s).
struct NormGrad {
    const void *dh, *dn;                                     // either may be NULL
    const float *stats;
    void *dy, *d_residual, *d_token;                         // any may be NULL; d_token: the per-token gate's gradient
    float *partial;
    int want_z, want_v;
};

// A vector over the channels lies in LDS as two halves, the first and the last four of every piece of eight: neighbouring
// lanes then read neighbouring 16 bytes.  (Pieces of 32 bytes back to back cost a bank conflict on every read: 1.5e8
// cycles over the card in a gradient of 16384 rows of 7168.  The halves read float by float still cost 4.4e7; as whole
// 16 bytes 1e5, at the same time within the noise, 278-284 us and 280-281.)
__device__ __forceinline__ int lds_slot(int c, int padded) { return (c & 4 ? padded / 2 : 0) + c / 8 * 4 + c % 4; }

template <int E>
__device__ __forceinline__ void take_channels(bool given, const float *lds, int padded, int at, int tpr, float fill, float *f) {
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        const int c = (at + i * tpr) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i * 8 + j] = fill;
        if (given && c < padded) {                           // whole pieces: the LDS rows are padded to them
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f32x4 v = *(const f32x4 *)(lds + lds_slot(c, padded) + j * (padded / 2));
#pragma unroll
                for (int k = 0; k < 4; ++k) f[i * 8 + j * 4 + k] = v[k];
            }
        }
    }
}

template <int TY, int TR, bool ALIGNED, int E, bool WIDE, bool DN>
__global__ __launch_bounds__(kNormThreads) void block_norm_grad_kernel(NormArgs a, NormGrad d) {
    __shared__ float part[2][kNormWaves * 3];
    extern __shared__ __align__(16) float vectors[];         // [2][H up to a piece]: w_post * gate, w_pre
    const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.x / a.tpr);          // whole waves per row
    const int at = (int)threadIdx.x - group * a.tpr;
    const float inv_h = 1.0f / (float)a.H;
    const int64_t stride = (int64_t)gridDim.x * a.groups;
    const void *channel_gate = a.gate_kind == TERRACE_GATE_CHANNEL ? a.gate : nullptr;
    const int padded = (int)((a.H + 7) / 8 * 8);
    const bool has_b = a.w_post || channel_gate, need_y = a.y && (DN || a.w_post || a.gate);
    const bool need_dot = a.w_post || d.d_token;
    float *lds_b = vectors, *lds_pre = vectors + padded;
    if constexpr (!WIDE) {
        for (int c = threadIdx.x; c < padded; c += blockDim.x) {
            const bool in = c < a.H;
            float b = in ? 1.0f : 0.0f;
            if (a.w_post && in) b *= load_scalar(a.w_post, a.post_dtype, c);
            if (channel_gate && in) b *= load_scalar(channel_gate, a.gate_dtype, c);
            if (has_b) lds_b[lds_slot(c, padded)] = b;
            if (DN) lds_pre[lds_slot(c, padded)] = in ? load_scalar(a.w_pre, a.pre_dtype, c) : 0.0f;
        }
        __syncthreads();
    }
    // the vectors of this lane's channels: w_post times the gate per channel (the only way they come in), and w_pre
    auto take = [&](float *b, float *wn) {
        if constexpr (WIDE) {
            float g[E];
            load_channels<ALIGNED, E>(a.w_post, a.post_dtype, a.H, at, a.tpr, 1.0f, b);
            load_channels<ALIGNED, E>(channel_gate, a.gate_dtype, a.H, at, a.tpr, 1.0f, g);
            if constexpr (DN) load_channels<ALIGNED, E>(a.w_pre, a.pre_dtype, a.H, at, a.tpr, 0.0f, wn);
#pragma unroll
            for (int e = 0; e < E; ++e) b[e] *= g[e];
        } else {
            take_channels<E>(has_b, lds_b, padded, at, a.tpr, 1.0f, b);
            if constexpr (DN) take_channels<E>(true, lds_pre, padded, at, a.tpr, 0.0f, wn);
        }
    };
    float sum[2][WIDE ? 1 : E];
    if constexpr (!WIDE) {
#pragma unroll
        for (int e = 0; e < E; ++e) sum[0][e] = sum[1][e] = 0.0f;
    }
    struct Row {
        Share<TY, ALIGNED, E> y, dn;
        Share<TR, ALIGNED, E> r, dh;
        float inv1, inv2, token;
    };
    auto fetch = [&](int64_t row, Row &x) {
        x.y.clear(), x.r.clear(), x.dh.clear(), x.dn.clear();
        x.inv1 = x.inv2 = x.token = 1.0f;
        if (row >= a.T) return;
        if (need_y) x.y.load(a.y, row, a.H, at, a.tpr);
        if constexpr (DN) x.r.load(a.residual, row, a.H, at, a.tpr);
        if (d.dh) x.dh.load(d.dh, row, a.H, at, a.tpr);
        if constexpr (DN) x.dn.load(d.dn, row, a.H, at, a.tpr);
        x.inv1 = d.stats[2 * row];
        if constexpr (DN) x.inv2 = d.stats[2 * row + 1];
        if (a.gate_kind == TERRACE_GATE_TOKEN) x.token = load_scalar(a.gate, a.gate_dtype, row);
    };
    const int64_t first = (int64_t)blockIdx.x * a.groups;
    Row cur, next;
    fetch(first + group, cur);
    int turn = 0;
    for (int64_t base = first; base < a.T; base += stride) {
        const int64_t row = base + group;
        const bool mine = row < a.T;
        if constexpr (!WIDE) fetch(row + stride, next);
        const float factor = a.scale * cur.token;            // scale, and the token's gate where there is one
        float b[E], wn[E];
        take(b, wn);
        float mean_tv = 0.0f, dot;                           // dot: sum of dH * gate per channel * p
        if constexpr (DN) {
            float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float u = cur.y.get(e) * cur.inv1, q = u * b[e];
                const float h = __fmaf_rn(factor, q, cur.r.get(e)), v = h * cur.inv2, t = cur.dn.get(e) * wn[e];
                s[0] = __fmaf_rn(t, v, s[0]);
                s[1] = __fmaf_rn(__fmaf_rn(cur.inv2, t, cur.dh.get(e)), q, s[1]);
                s[2] = __fmaf_rn(v, q, s[2]);
            }
            row_sum<3>(s, part[turn], a.tpr);
            mean_tv = s[0] * inv_h;
            dot = __fmaf_rn(-cur.inv2 * mean_tv, s[2], s[1]);
        } else {
            dot = 0.0f;
            if (need_dot) {
#pragma unroll
                for (int e = 0; e < E; ++e) dot = __fmaf_rn(cur.dh.get(e), cur.y.get(e) * cur.inv1 * b[e], dot);
                row_sum<1>(&dot, part[turn], a.tpr);
            }
        }
        turn ^= 1;
        const float mean_u = factor * dot * inv_h;
        take(b, wn);
        float o1[E], o2[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float u = cur.y.get(e) * cur.inv1;
            float v = 0.0f, dn = 0.0f, dH = cur.dh.get(e);
            if constexpr (DN) {
                v = __fmaf_rn(factor, u * b[e], cur.r.get(e)) * cur.inv2;
                dn = cur.dn.get(e);
                dH = __fmaf_rn(cur.inv2, __fmaf_rn(-v, mean_tv, dn * wn[e]), dH);
            }
            const float z = factor * dH;
            o1[e] = dH;
            o2[e] = z * b[e];
            if (a.w_post) o2[e] = cur.inv1 * __fmaf_rn(-u, mean_u, o2[e]);
            if constexpr (!WIDE) {
                sum[0][e] = __fmaf_rn(z, u, sum[0][e]);
                if constexpr (DN) sum[1][e] = __fmaf_rn(dn, v, sum[1][e]);
            } else if (mine) {                               // one group: this lane alone touches the channel's cells
                const int64_t c = ((int64_t)at + (int64_t)(e / 8) * a.tpr) * 8 + e % 8;
                if (c < a.H) {
                    float *cell = d.partial + (int64_t)blockIdx.x * a.H + c;
                    if (d.want_z) *cell = base == first ? z * u : __fmaf_rn(z, u, *cell);
                    cell += (int64_t)gridDim.x * a.H;
                    if (d.want_v) *cell = base == first ? dn * v : __fmaf_rn(dn, v, *cell);
                }
            }
        }
        if (mine) {
            if (d.d_residual) store_share<TR, ALIGNED, E>(d.d_residual, row, a.H, at, a.tpr, o1);
            if (d.dy) store_share<TY, ALIGNED, E>(d.dy, row, a.H, at, a.tpr, o2);
            if (d.d_token && at == 0) {
                const float dg = a.scale * dot;
                if (a.gate_dtype == TERRACE_F32) store_floats<TERRACE_F32, 1>(d.d_token, row, &dg);
                else if (a.gate_dtype == TERRACE_BF16) store_floats<TERRACE_BF16, 1>(d.d_token, row, &dg);
                else store_floats<TERRACE_F16, 1>(d.d_token, row, &dg);
            }
        }
        if constexpr (WIDE) fetch(row + stride, cur);
        else cur = next;
    }
    if constexpr (!WIDE) {
        const int want[2] = {d.want_z, d.want_v};
        __syncthreads();                                     // the vectors' LDS holds the joined sums from here on
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (!want[k]) continue;
            float *out = d.partial + ((int64_t)k * gridDim.x + blockIdx.x) * a.H;
            if (a.groups == 1) {
                store_share<TERRACE_F32, ALIGNED, E>(out, 0, a.H, at, a.tpr, sum[k]);
                continue;
            }
            for (int g = 0; g < a.groups; ++g) {             // the row groups one after the other: a fixed order
                if (group == g) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int c = (at + (e / 8) * a.tpr) * 8 + e % 8;
                        if (c < a.H) vectors[c] = g ? vectors[c] + sum[k][e] : sum[k][e];
                    }
                }
                __syncthreads();
            }
            for (int64_t c = threadIdx.x; c < a.H; c += blockDim.x) out[c] = vectors[c];
            __syncthreads();
        }
    }
}

// The workgroups' partial rows added up, 64 columns a workgroup: its 16 waves take every 16th partial row and are joined
// in order.  blockIdx.y = 0: sum(factor dH u), which times the gate is d_w_post and times w_post is the gradient of a
// gate per channel; 1: d_w_pre.
struct NormReduce {
    void *d_post, *d_gate, *d_pre;
};
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float *__restrict__ partial, int rows, NormArgs a,
                                                           NormReduce r) {
    __shared__ float part[16][kWave];
    const int k = blockIdx.y, w = wave_in_block(), lane = lane_id();
    if (k == 0 ? !r.d_post && !r.d_gate : !r.d_pre) return;
    const int64_t c = (int64_t)blockIdx.x * kWave + lane;
    const float *p = partial + (int64_t)k * rows * a.H;
    float v = 0.0f;
    if (c < a.H) {
#pragma unroll 8
        for (int g = w; g < rows; g += 16) v += p[(int64_t)g * a.H + c];
    }
    part[w][lane] = v;
    __syncthreads();
    if (w || c >= a.H) return;
    v = 0.0f;
#pragma unroll
    for (int x = 0; x < 16; ++x) v += part[x][lane];
    auto put = [&](void *out, int dtype, float f) {
        if (dtype == TERRACE_F32) store_floats<TERRACE_F32, 1>(out, c, &f);
        else if (dtype == TERRACE_BF16) store_floats<TERRACE_BF16, 1>(out, c, &f);
        else store_floats<TERRACE_F16, 1>(out, c, &f);
    };
    if (k == 1) {
        put(r.d_pre, a.pre_dtype, v);
        return;
    }
    if (r.d_post) put(r.d_post, a.post_dtype, a.gate_kind == TERRACE_GATE_CHANNEL ? v * load_scalar(a.gate, a.gate_dtype, c) : v);
    if (r.d_gate) put(r.d_gate, a.gate_dtype, a.w_post ? v * load_scalar(a.w_post, a.post_dtype, c) : v);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr int64_t kNormMaxH = 2 * 8 * kNormThreads;          // 16 elements a lane
constexpr int kNormBlocks = 256;                             // one workgroup a CU (two: 182 us where one takes 173)
constexpr int kNormGradBlocks = 256;

static bool norm_float(int d) { return d == TERRACE_F32 || d == TERRACE_BF16 || d == TERRACE_F16; }

// Elements a lane holds, and whether the rows are whole pieces on 16-byte boundaries (otherwise any alignment their
// elements have).
struct NormForm {
    int per;
    bool aligned;
};
static NormForm norm_form(const NormArgs &a, uintptr_t bits) {
    return {a.H <= kNormMaxH / 2 ? 8 : 16, a.H % 8 == 0 && (bits & 15) == 0};
}

static int norm_check(const NormArgs &a, int y_dtype, int r_dtype) {
    if (a.T < 0 || a.H <= 0 || a.H > kNormMaxH || !norm_float(y_dtype) || !norm_float(r_dtype) ||
        (r_dtype != y_dtype && r_dtype != TERRACE_F32) || a.gate_kind < TERRACE_GATE_NONE || a.gate_kind > TERRACE_GATE_TOKEN ||
        (a.T > 0 && (a.gate_kind != TERRACE_GATE_NONE) != (a.gate != nullptr)) || (a.w_post && !norm_float(a.post_dtype)) ||
        (a.gate && !norm_float(a.gate_dtype)) || (a.w_pre && !norm_float(a.pre_dtype)) ||
        (a.T > 0 && !a.y && (a.w_post || a.gate)))
        return TERRACE_EINVAL;
    return TERRACE_OK;
}

static void norm_shape(NormArgs &a, int per) {
    a.tpr = (int)(((a.H + per - 1) / per + kWave - 1) / kWave * kWave);
    a.groups = 1;
}

// Rows a workgroup works on at a time: as many as it has threads for, but no more than leave every CU a workgroup.
static void norm_groups(NormArgs &a) {
    const int64_t most = kNormThreads / a.tpr, even = a.T / 256;
    a.groups = (int)(even < 1 ? 1 : even < most ? even : most);
}

#define TERRACE_NORM_TYPES(CALL)                                                                  \
    if (y_dtype == TERRACE_F32) { CALL(TERRACE_F32, TERRACE_F32); }                               \
    else if (y_dtype == TERRACE_BF16 && r_dtype == TERRACE_BF16) { CALL(TERRACE_BF16, TERRACE_BF16); } \
    else if (y_dtype == TERRACE_BF16) { CALL(TERRACE_BF16, TERRACE_F32); }                        \
    else if (r_dtype == TERRACE_F16) { CALL(TERRACE_F16, TERRACE_F16); }                          \
    else { CALL(TERRACE_F16, TERRACE_F32); }

int run_block_norm(const void *y, int y_dtype, const void *residual, int r_dtype, const void *w_post, int post_dtype,
                   const void *gate, int gate_dtype, int gate_kind, const void *w_pre, int pre_dtype, float scale,
                   float eps, int64_t T, int64_t H, void *h, void *n, float *stats, hipStream_t s) {
    NormArgs a{y, residual, w_post, gate, w_pre, post_dtype, gate_dtype, pre_dtype, gate_kind, scale, eps, T, H, 0, 1};
    int rc = norm_check(a, y_dtype, r_dtype);
    if (rc != TERRACE_OK) return rc;
    uintptr_t bits = (uintptr_t)y | (uintptr_t)residual | (uintptr_t)w_post | (uintptr_t)w_pre | (uintptr_t)h | (uintptr_t)n;
    if (gate_kind == TERRACE_GATE_CHANNEL) bits |= (uintptr_t)gate;
    const NormForm form = norm_form(a, bits);
    if (T == 0) return TERRACE_OK;
    if (!residual || (y && !h) || (w_pre && !n)) return TERRACE_EINVAL;
    norm_shape(a, form.per);
    norm_groups(a);
    const int64_t need = (T + a.groups - 1) / a.groups;
    const unsigned grid = (unsigned)(need < kNormBlocks ? need : kNormBlocks), threads = (unsigned)(a.tpr * a.groups);
#define TERRACE_NORM_AHEAD(Y, R, A, E)                                                                     \
    if (norm_two_ahead(R, A, E) && need > 8 * kNormBlocks)                                                 \
        block_norm_kernel<Y, R, A, E, norm_two_ahead(R, A, E) ? 2 : 1><<<grid, threads, 0, s>>>(a, h, n, stats); \
    else block_norm_kernel<Y, R, A, E, 1><<<grid, threads, 0, s>>>(a, h, n, stats)
#define TERRACE_NORM(Y, R)                                                     \
    if (form.aligned && form.per == 8) { TERRACE_NORM_AHEAD(Y, R, true, 8); }  \
    else if (form.aligned) { TERRACE_NORM_AHEAD(Y, R, true, 16); }             \
    else if (form.per == 8) { TERRACE_NORM_AHEAD(Y, R, false, 8); }            \
    else { TERRACE_NORM_AHEAD(Y, R, false, 16); }
    TERRACE_NORM_TYPES(TERRACE_NORM)
#undef TERRACE_NORM
#undef TERRACE_NORM_AHEAD
    return check_launch();
}

static unsigned norm_grad_grid(int64_t T, int groups) {
    const int64_t need = (T + groups - 1) / groups;
    return (unsigned)(need < kNormGradBlocks ? need : kNormGradBlocks);
}

size_t block_norm_grad_workspace(int64_t T, int64_t H) {
    if (T <= 0 || H <= 0 || H > kNormMaxH) return 256;
    const int64_t grid = T < kNormGradBlocks ? T : kNormGradBlocks;
    return align_up((size_t)(2 * grid * H) * sizeof(float), 256);
}

int run_block_norm_grad(const void *y, int y_dtype, const void *residual, int r_dtype, const void *w_post,
                        int post_dtype, const void *gate, int gate_dtype, int gate_kind, const void *w_pre,
                        int pre_dtype, float scale, float eps, int64_t T, int64_t H, const float *stats, const void *dh,
                        const void *dn, void *dy, void *d_residual, void *d_post, void *d_gate, void *d_pre, void *ws,
                        size_t ws_bytes, hipStream_t s) {
    NormArgs a{y, residual, w_post, gate, w_pre, post_dtype, gate_dtype, pre_dtype, gate_kind, scale, eps, T, H, 0, 1};
    int rc = norm_check(a, y_dtype, r_dtype);
    if (rc != TERRACE_OK) return rc;
    if ((d_post && !w_post) || (T > 0 && d_gate && !gate) || (d_pre && !w_pre) || (T > 0 && dy && !y) || (dn && !w_pre))
        return TERRACE_EINVAL;
    uintptr_t bits = (uintptr_t)y | (uintptr_t)residual | (uintptr_t)w_post | (uintptr_t)w_pre | (uintptr_t)dh |
                     (uintptr_t)dn | (uintptr_t)dy | (uintptr_t)d_residual | (uintptr_t)ws;
    if (gate_kind == TERRACE_GATE_CHANNEL) bits |= (uintptr_t)gate;
    const NormForm form = norm_form(a, bits);
    if ((uintptr_t)ws & 15) return TERRACE_EINVAL;
    const bool channel_gate = gate_kind == TERRACE_GATE_CHANNEL;
    const NormReduce red{d_post, channel_gate ? d_gate : nullptr, d_pre};
    const bool want_z = red.d_post || red.d_gate, want_v = red.d_pre != nullptr, sums = want_z || want_v;
    if (sums && (!ws || ws_bytes < block_norm_grad_workspace(T, H))) return ws ? TERRACE_ENOSPC : TERRACE_EINVAL;
    unsigned grid = 0;
    if (T > 0) {
        if (!residual || !stats) return TERRACE_EINVAL;
        norm_shape(a, form.per);
        if (form.per == 8) norm_groups(a);
        grid = norm_grad_grid(T, a.groups);
        const NormGrad d{dh, dn, stats, dy, d_residual, gate_kind == TERRACE_GATE_TOKEN ? d_gate : nullptr, (float *)ws, want_z,
                         want_v};
        const unsigned threads = (unsigned)(a.tpr * a.groups);
        const size_t lds = form.per == 16 ? 0 : (size_t)(2 * ((H + 7) / 8 * 8)) * sizeof(float);
#define TERRACE_NORM_FORM(Y, R, A, E, WIDE)                                                                     \
    if (dn) block_norm_grad_kernel<Y, R, A, E, WIDE, true><<<grid, threads, lds, s>>>(a, d);                   \
    else block_norm_grad_kernel<Y, R, A, E, WIDE, false><<<grid, threads, lds, s>>>(a, d)
#define TERRACE_NORM(Y, R)                                                               \
    if (form.aligned && form.per == 8) { TERRACE_NORM_FORM(Y, R, true, 8, false); }      \
    else if (form.aligned) { TERRACE_NORM_FORM(Y, R, true, 16, true); }                  \
    else if (form.per == 8) { TERRACE_NORM_FORM(Y, R, false, 8, false); }                \
    else { TERRACE_NORM_FORM(Y, R, false, 16, true); }
        TERRACE_NORM_TYPES(TERRACE_NORM)
#undef TERRACE_NORM
#undef TERRACE_NORM_FORM
    }
    if (sums)
        norm_reduce_kernel<<<dim3((unsigned)((H + kWave - 1) / kWave), 2), 1024, 0, s>>>((const float *)ws, (int)grid, a, red);
    return check_launch();
}

}  // namespace terrace
