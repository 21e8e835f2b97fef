// Tokens to expert order and back without the hops between: the (token, expert) pairs of a routing sorted by expert,
// the rows moved there, and the gradient of the weighted way back.
//
//   expert_sort_small_kernel  few pairs: one launch that ranks, counts and moves
//   expert_tail_kernel        zero rows behind the live ones (the index comes from sort.hip, the rows move with the
//                             scatter of rows.hip)
//   expert_unsort_grad_kernel d_rows[where[t,j]] = w[t,j] * dy[t],  d_weights[t,j] = <dy[t], rows[where[t,j]]>
//
// The way back itself is the combine of rows.hip, and the gradient of the sort is the combine without weights.
#include "sort.hpp"

namespace terrace {

size_t expert_index_workspace(int64_t P, int n_experts);
int run_expert_index(const int64_t *expert_idx, int64_t P, int n_experts, int64_t *where, int64_t *tokens_per_expert,
                     int64_t *offsets, int32_t *status, void *ws, const int32_t **pos32, const int32_t **live,
                     hipStream_t s);

// ---------------------------------------------------------------------------------------------
// few pairs: one launch
// ---------------------------------------------------------------------------------------------
// With few pairs the place of a pair is found by comparing it with every other one: with key(p) = expert of p
// (n_experts for a pair without one) and code(p) = key(p) * P + p, place(p) = #{p' : code(p') < code(p)}.  Every
// workgroup does that for the k pairs of its own token -- P * k compares, one ballot per 64 of them -- and then moves its
// slice of the token's row; a pair without an expert ranks behind all others, so its place is one of the rows behind
// the live ones and the workgroup writes zeros there.  The last workgroup writes the counts.  No workspace, no second
// launch: what bounds it is the latency of one launch and two dependent reads (the ids, then nothing but stores).
// 8 experts of 256 a token, 14 KB rows, against the sorting path: 32 tokens 4.7 us for 9.8, 128 tokens 7.9 for 10.9, 512
// tokens 26 for 35, 1024 tokens 62 for 48; one expert a token, 2000 tokens 10.3 for 19.2, 8000 tokens 66 for 17.
//
// Every workgroup of a token repeats its ranking, and a row in pieces of a few bytes (an odd width, a base off 16 bytes) has
// many slices: 28 at 7167 bf16.  So a token gets no more workgroups than 2048 in all need, but four, and each walks on over
// the row: 512 such tokens 43 us, 111 with a workgroup a slice, where 513 take the sorting path in 53; 2000 tokens of one
// expert 49 us for 170 (2049: 72); 16 tokens 5.9 us either way.
static bool few_pairs(int64_t T, int64_t P) { return P <= 2048 || (P <= 4096 && T <= 1024); }
constexpr int kMaxSmallExperts = kMaxBuckets;
constexpr int kSmallFan = 16;
constexpr int kSmallGroups = 2048;

template <typename V>
__global__ __launch_bounds__(kBlock) void expert_sort_small_kernel(
    const V *__restrict__ x, const int64_t *__restrict__ expert_idx, int T, int k, int n_experts, int64_t row_vecs,
    int64_t live_vecs, int slices, V *__restrict__ rows, int64_t *__restrict__ where,
    int64_t *__restrict__ tokens_per_expert, int64_t *__restrict__ offsets, int32_t *__restrict__ status) {
    __shared__ int32_t counts[kMaxSmallExperts + 1];
    __shared__ int32_t below[kWavesPerBlock][kSmallFan];
    __shared__ int32_t faults;
    const int lane = lane_id(), w = wave_in_block(), P = T * k;
    if ((int)blockIdx.x == T * slices) {                     // counts, offsets, status
        for (int e = threadIdx.x; e <= n_experts; e += kBlock) counts[e] = 0;
        if (threadIdx.x == 0) faults = 0;
        __syncthreads();
        for (int p = threadIdx.x; p < P; p += kBlock) {
            const int64_t id = expert_idx[p];
            if (id >= 0 && id < n_experts) atomicAdd(&counts[(int)id], 1);
            else if (id >= n_experts) atomicOr(&faults, TERRACE_FAULT_ID_RANGE);
        }
        __syncthreads();
        if (w == 0) {
            int carry = 0;
            for (int e0 = 0; e0 < n_experts; e0 += kWave) {
                const int e = e0 + lane;
                const int v = e < n_experts ? counts[e] : 0;
                const int incl = wave_inclusive_scan(v);
                if (e < n_experts) {
                    tokens_per_expert[e] = v;
                    offsets[e] = carry + incl - v;
                }
                carry += __shfl(incl, kWave - 1, kWave);
            }
            if (lane == 0) offsets[n_experts] = carry;
            if (lane < TERRACE_STATUS_WORDS && status) status[lane] = lane == 0 ? faults : 0;
        }
        return;
    }
    const int t = (int)blockIdx.x / slices, slice = (int)blockIdx.x - t * slices;
    const int64_t i = (int64_t)slice * kBlock + threadIdx.x, step = (int64_t)slices * kBlock;
    V v = zero_of<V>();
    if (rows && i < live_vecs) v = x[(int64_t)t * row_vecs + i];
    for (int j0 = 0; j0 < k; j0 += kSmallFan) {              // one round for k <= 16
        const int m = k - j0 < kSmallFan ? k - j0 : kSmallFan;
        // lane j < m holds its pair's code; the loop below broadcasts them
        int64_t id = -1;
        if (lane < m) id = expert_idx[t * k + j0 + lane];
        const int key = id >= 0 && id < n_experts ? (int)id : n_experts;
        const int code = key * P + t * k + j0 + lane;
        int n[kSmallFan];
#pragma unroll
        for (int j = 0; j < kSmallFan; ++j) n[j] = 0;
        for (int p0 = w * kWave; p0 < P; p0 += kBlock) {
            const int p = p0 + lane;
            int other = 0x7FFFFFFF;
            if (p < P) {
                const int64_t o = expert_idx[p];
                other = (o >= 0 && o < n_experts ? (int)o : n_experts) * P + p;
            }
#pragma unroll
            for (int j = 0; j < kSmallFan; ++j) {
                if (j < m) n[j] += __popcll(__ballot(other < read_lane(code, j)));
            }
        }
#pragma unroll
        for (int j = 0; j < kSmallFan; ++j) {
            if (lane == j) below[w][j] = n[j];
        }
        __syncthreads();
        const uint64_t alive = __ballot(key < n_experts);
        if (slice == 0 && w == 0 && lane < m)
            where[t * k + j0 + lane] = alive >> lane & 1 ? below[0][lane] + below[1][lane] + below[2][lane] + below[3][lane] : -1;
        V u = v;
        for (int64_t c = i; rows && c < live_vecs; c += step) {          // once where the slices are the whole row
            if (c != i) u = x[(int64_t)t * row_vecs + c];
            for (int j = 0; j < m; ++j) {
                const int place = below[0][j] + below[1][j] + below[2][j] + below[3][j];
                rows[(int64_t)place * row_vecs + c] = alive >> j & 1 ? u : zero_of<V>();
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// zero rows behind the live ones
// ---------------------------------------------------------------------------------------------
constexpr int kTailBlocks = 1024;

template <typename V>
__global__ __launch_bounds__(kBlock) void expert_tail_kernel(const int32_t *__restrict__ live, int64_t P,
                                                             V *__restrict__ rows, int64_t row_vecs, int64_t live_vecs,
                                                             int64_t *__restrict__ total) {
    const int64_t first = *live;
    if (blockIdx.x == 0 && threadIdx.x == 0) *total = first;
    if (!rows) return;
    for (int64_t r = first + blockIdx.x; r < P; r += gridDim.x)
        for (int64_t i = threadIdx.x; i < live_vecs; i += kBlock) rows[r * row_vecs + i] = zero_of<V>();
}

__global__ __launch_bounds__(kBlock) void expert_empty_kernel(int64_t *__restrict__ tokens_per_expert,
                                                              int64_t *__restrict__ offsets, int n_experts,
                                                              int32_t *__restrict__ status) {
    for (int e = threadIdx.x; e <= n_experts; e += kBlock) {
        if (e < n_experts) tokens_per_expert[e] = 0;
        offsets[e] = 0;
    }
    if (status && threadIdx.x < TERRACE_STATUS_WORDS) status[threadIdx.x] = 0;
}

static int row_vec_bytes(const RowGeom &g, const void *a, const void *b) {
    const uintptr_t bits = (uintptr_t)g.width | (uintptr_t)g.pitch | (uintptr_t)a | (uintptr_t)b;
    return (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1;
}

size_t expert_sort_workspace(int64_t T, int k, int n_experts) {
    if (T <= 0 || k <= 0 || T > (((int64_t)1 << 31) - 1) / k || few_pairs(T, T * k)) return 256;
    return expert_index_workspace(T * k, n_experts);
}

int run_expert_sort(const void *x, const int64_t *expert_idx, int64_t T, int64_t row_bytes, int k, int n_experts,
                    void *rows, int64_t *where, int64_t *tokens_per_expert, int64_t *offsets, int32_t *status, void *ws,
                    size_t ws_bytes, hipStream_t s) {
    const RowGeom g = row_geom(row_bytes);
    if (T < 0 || k <= 0 || n_experts <= 0 || n_experts > kMaxBuckets || row_bytes < 0 || !row_geom_ok(g) ||
        !tokens_per_expert || !offsets || T > (((int64_t)1 << 31) - 1) / k)
        return TERRACE_EINVAL;
    const int64_t P = T * k;
    if (P == 0) {
        expert_empty_kernel<<<1, kBlock, 0, s>>>(tokens_per_expert, offsets, n_experts, status);
        return check_launch();
    }
    if (!expert_idx || !where || (x != nullptr) != (rows != nullptr)) return TERRACE_EINVAL;
    if (x && g.pitched() && (((uintptr_t)x | (uintptr_t)rows) & 15)) return TERRACE_EINVAL;
    const bool move = x && g.width > 0;
    const int vb = move ? row_vec_bytes(g, x, rows) : 16;
    if (few_pairs(T, P)) {
        const int64_t vecs = move ? g.width / vb : 1, most = kSmallGroups / T > 4 ? kSmallGroups / T : 4;
        const int64_t need = (vecs + kBlock - 1) / kBlock, slices = need < most ? need : most;
        const unsigned grid = (unsigned)(T * slices + 1);
#define TERRACE_SMALL(V)                                                                                            \
    expert_sort_small_kernel<V><<<grid, kBlock, 0, s>>>((const V *)x, expert_idx, (int)T, k, n_experts, g.pitch / vb, \
                                                        vecs, (int)slices, move ? (V *)rows : nullptr, where,        \
                                                        tokens_per_expert, offsets, status)
        if (vb == 16) TERRACE_SMALL(u32x4);
        else if (vb == 4) TERRACE_SMALL(uint32_t);
        else if (vb == 2) TERRACE_SMALL(uint16_t);
        else TERRACE_SMALL(uint8_t);
#undef TERRACE_SMALL
        return check_launch();
    }
    if (!ws) return TERRACE_EINVAL;
    if (ws_bytes < expert_sort_workspace(T, k, n_experts)) return TERRACE_ENOSPC;
    const int32_t *pos32 = nullptr, *live = nullptr;
    int rc = run_expert_index(expert_idx, P, n_experts, where, tokens_per_expert, offsets, status, ws, &pos32, &live, s);
    if (rc != TERRACE_OK) return rc;
    const unsigned grid = (unsigned)(P < kTailBlocks ? P : kTailBlocks);
#define TERRACE_TAIL(V)                                                                                           \
    expert_tail_kernel<V><<<grid, kBlock, 0, s>>>(live, P, move ? (V *)rows : nullptr, g.pitch / vb, g.width / vb, \
                                                  offsets + n_experts)
    if (vb == 16) TERRACE_TAIL(u32x4);
    else if (vb == 4) TERRACE_TAIL(uint32_t);
    else if (vb == 2) TERRACE_TAIL(uint16_t);
    else TERRACE_TAIL(uint8_t);
#undef TERRACE_TAIL
    rc = check_launch();
    if (rc != TERRACE_OK || !move) return rc;
    return launch_scatter_rows<int32_t>(x, rows, pos32, T, k, row_bytes, P, s);
}

// ---------------------------------------------------------------------------------------------
// gradient of the weighted way back
// ---------------------------------------------------------------------------------------------
// One workgroup per token: the row of dy is read once and stays in registers while the token's k rows are read beside
// it, k scaled copies of it are written and k dot products are summed, all in one pass, so the launch moves (1 + 2k)
// rows per token and nothing twice.  Products and sums are fp32; a lane adds its own chunks in ascending order, the
// lanes are joined by a butterfly and the waves in order, so the result does not depend on timing.  Rows from
// offsets[n_experts] on belong to no pair: the workgroups past the tokens write them as zeros.
//
// What bounds it is the memory system under k + 1 read and k write streams of rows at scattered places: 16384 tokens x 8
// rows of 14 KB, 3.99 GB in 780 us, 5.1 TB/s, the same within 1 % for 1, 2, 4 or 7 waves a token and for 32 down to 12
// resident waves a CU (4: 808 us).  Place by place -- both large arrays in order, dy read k times -- it took 877-1056 us.  A
// width that is no multiple of 8, or a base off 16 bytes, goes element by element: 7167 in the place of 7168 1020 us.
constexpr int kGradFan = 8;

// N elements of a row as they were loaded: eight rows of pieces wait in registers, and unpacked they would take twice
// the registers.
template <int DT, int N>
struct Piece {
    static constexpr int kWords = N == 1 ? 1 : DT == TERRACE_F32 ? 8 : 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const uint8_t *row, int64_t c) {
        if constexpr (N == 1) {
            if constexpr (DT == TERRACE_F32) w[0] = ((const uint32_t *)row)[c];
            else w[0] = ((const uint16_t *)row)[c];
        } else {
#pragma unroll
            for (int v = 0; v < kWords / 4; ++v) {
                const u32x4 x = ld_stream((const u32x4 *)row + c * (kWords / 4) + v);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * v + i] = x[i];
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == TERRACE_F32) {
            return __uint_as_float(w[i]);
        } else {
            const uint32_t b = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
            if constexpr (DT == TERRACE_BF16) return bf16_bits_to_f32(b);
            else return __half2float(__ushort_as_half((unsigned short)b));
        }
    }
};

template <int SRC, int DY, int N>
__global__ __launch_bounds__(kBlock) void expert_unsort_grad_kernel(
    const uint8_t *__restrict__ src, const uint8_t *__restrict__ dy, const int64_t *__restrict__ where,
    const void *__restrict__ weights, int w_dtype, int64_t T, int k, int64_t hidden, int64_t n_rows,
    const int64_t *__restrict__ live, uint8_t *__restrict__ d_rows, void *__restrict__ d_weights) {
    constexpr int64_t kSrcBytes = SRC == TERRACE_F32 ? 4 : 2, kDyBytes = DY == TERRACE_F32 ? 4 : 2;
    __shared__ float part[kWavesPerBlock][kGradFan];
    const int64_t chunks = hidden / N;
    if ((int64_t)blockIdx.x >= T) {
        if (!d_rows) return;
        const float zeros[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        int64_t first = *live;
        if (first < 0) first = 0;
        for (int64_t r = first + (blockIdx.x - T); r < n_rows; r += gridDim.x - T)
            for (int64_t c = threadIdx.x; c < chunks; c += blockDim.x)
                store_floats<SRC, N>(d_rows + r * hidden * kSrcBytes, c * N, zeros);
        return;
    }
    const int64_t t = blockIdx.x;
    const uint8_t *dy_row = dy + t * hidden * kDyBytes;
    const int waves = (int)(blockDim.x >> 6);
    for (int j0 = 0; j0 < k; j0 += kGradFan) {               // one round for k <= 8
        const int m = k - j0 < kGradFan ? k - j0 : kGradFan;
        int64_t at[kGradFan];
        float w[kGradFan], sum[kGradFan];
#pragma unroll
        for (int j = 0; j < kGradFan; ++j) {
            at[j] = -1;
            w[j] = 1.0f;
            sum[j] = 0.0f;
            if (j < m) {
                const int64_t p = t * k + j0 + j;
                at[j] = where[p];
                if (!row_in(at[j], n_rows)) at[j] = -1;
                if (weights) {
                    if (w_dtype == TERRACE_F32) load_floats<TERRACE_F32, 1>(weights, p, &w[j]);
                    else if (w_dtype == TERRACE_BF16) load_floats<TERRACE_BF16, 1>(weights, p, &w[j]);
                    else load_floats<TERRACE_F16, 1>(weights, p, &w[j]);
                }
            }
        }
        for (int64_t c = threadIdx.x; c < chunks; c += blockDim.x) {
            Piece<SRC, N> f[kGradFan];
            Piece<DY, N> gp;
            gp.load(dy_row, c);
            if (d_weights) {
#pragma unroll
                for (int j = 0; j < kGradFan; ++j) {
                    if (at[j] >= 0) f[j].load(src + at[j] * hidden * kSrcBytes, c);
                }
            }
            float g[N];
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = gp.get(i);
            if (d_weights) {
#pragma unroll
                for (int j = 0; j < kGradFan; ++j) {
                    if (at[j] >= 0) {
#pragma unroll
                        for (int i = 0; i < N; ++i) sum[j] = __fmaf_rn(g[i], f[j].get(i), sum[j]);
                    }
                }
            }
            if (d_rows) {
#pragma unroll
                for (int j = 0; j < kGradFan; ++j) {
                    if (at[j] >= 0) {
                        float o[N];
#pragma unroll
                        for (int i = 0; i < N; ++i) o[i] = __fmul_rn(w[j], g[i]);
                        store_floats<SRC, N>(d_rows + at[j] * hidden * kSrcBytes, c * N, o);
                    }
                }
            }
        }
        if (!d_weights) continue;
#pragma unroll
        for (int j = 0; j < kGradFan; ++j) {
            const float v = wave_sum(sum[j]);
            if (lane_id() == 0) part[wave_in_block()][j] = v;
        }
        __syncthreads();
        if ((int)threadIdx.x < m) {
            float v = 0.0f;
            for (int x = 0; x < waves; ++x) v += part[x][threadIdx.x];
            const int64_t p = t * k + j0 + threadIdx.x;
            if (w_dtype == TERRACE_F32) store_floats<TERRACE_F32, 1>(d_weights, p, &v);
            else if (w_dtype == TERRACE_BF16) store_floats<TERRACE_BF16, 1>(d_weights, p, &v);
            else store_floats<TERRACE_F16, 1>(d_weights, p, &v);
        }
        __syncthreads();
    }
}

// Waves per token: the fewest rounds over the row that four waves allow, then no more waves than those rounds need.
static int grad_threads(int64_t chunks) {
    const int64_t waves = (chunks + kWave - 1) / kWave, rounds = (waves + kWavesPerBlock - 1) / kWavesPerBlock;
    return rounds ? (int)((waves + rounds - 1) / rounds) * kWave : kWave;
}

template <int SRC, int DY>
static void launch_unsort_grad(const void *src, const void *dy, const int64_t *where, const void *weights, int w_dtype,
                               int64_t T, int k, int64_t hidden, int64_t n_rows, const int64_t *live, void *d_rows,
                               void *d_weights, hipStream_t s) {
    const bool vec = hidden % 8 == 0 && (((uintptr_t)src | (uintptr_t)dy | (uintptr_t)d_rows) & 15) == 0;
    const int64_t chunks = vec ? hidden / 8 : hidden;
    const int threads = grad_threads(chunks);
    int64_t spare = n_rows < kTailBlocks ? n_rows : kTailBlocks;
    if (!d_rows) spare = 0;
    const unsigned grid = (unsigned)(T + spare);
    if (vec)
        expert_unsort_grad_kernel<SRC, DY, 8><<<grid, threads, 0, s>>>((const uint8_t *)src, (const uint8_t *)dy, where,
                                                                      weights, w_dtype, T, k, hidden, n_rows, live,
                                                                      (uint8_t *)d_rows, d_weights);
    else
        expert_unsort_grad_kernel<SRC, DY, 1><<<grid, threads, 0, s>>>((const uint8_t *)src, (const uint8_t *)dy, where,
                                                                      weights, w_dtype, T, k, hidden, n_rows, live,
                                                                      (uint8_t *)d_rows, d_weights);
}

int run_expert_unsort_grad(const void *src, int src_dtype, const void *dy, int dy_dtype, const int64_t *where,
                           const void *weights, int w_dtype, int64_t T, int k, int64_t hidden, int64_t n_rows,
                           const int64_t *live, void *d_rows, void *d_weights, hipStream_t s) {
    auto is_float = [](int d) { return d == TERRACE_F32 || d == TERRACE_BF16 || d == TERRACE_F16; };
    if (T < 0 || k <= 0 || hidden < 0 || n_rows < 0 || !is_float(src_dtype) || !is_float(dy_dtype) ||
        !is_float(w_dtype) || T > (((int64_t)1 << 31) - 1) / k || T + kTailBlocks >= ((int64_t)1 << 32) / kBlock)
        return TERRACE_EINVAL;                               // a launch has fewer than 2^32 threads
    if (!d_rows && !d_weights) return TERRACE_OK;
    if (T == 0 && n_rows == 0) return TERRACE_OK;
    if ((T && (!where || (hidden && (!dy || (d_weights && n_rows && !src))))) || (d_rows && !live)) return TERRACE_EINVAL;
#define TERRACE_GRAD(S, D) \
    launch_unsort_grad<S, D>(src, dy, where, weights, w_dtype, T, k, hidden, n_rows, live, d_rows, d_weights, s)
#define TERRACE_GRAD_S(S)                                            \
    if (dy_dtype == TERRACE_F32) TERRACE_GRAD(S, TERRACE_F32);       \
    else if (dy_dtype == TERRACE_BF16) TERRACE_GRAD(S, TERRACE_BF16); \
    else TERRACE_GRAD(S, TERRACE_F16)
    if (src_dtype == TERRACE_F32) { TERRACE_GRAD_S(TERRACE_F32); }
    else if (src_dtype == TERRACE_BF16) { TERRACE_GRAD_S(TERRACE_BF16); }
    else { TERRACE_GRAD_S(TERRACE_F16); }
#undef TERRACE_GRAD_S
#undef TERRACE_GRAD
    return check_launch();
}

}  // namespace terrace
