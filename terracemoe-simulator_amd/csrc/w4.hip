// The experts' products for a few rows each, on 4-bit weights with group scales.
//
//   w4_pack_kernel    codes, scales and zero points into the order the product reads them (once per weight)
//   w4_linear_kernel  out[i, n] = sum_k scale[e, n, k / g] * (code[e, n, k] - zero[e, n, k / g]) * x[i, k]
//                     for the rows i of expert e; optionally silu(first half of the columns) * (second half)
//
// Few rows per expert, so the product reads every code once and does little with it: it is bound by the HBM bytes of
// the weights of the experts that hold a row.  What the matrix cores are used for here is not their rate but that one
// instruction multiplies 8 codes of a lane with up to 16 rows.
#include "common.hpp"

namespace terrace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------
// packed layout
// ---------------------------------------------------------------------------------------------
// Codes: [experts][column tiles of 16][blocks of 128 k][64 lanes][4 dwords].  Lane l holds column l % 16 of its tile and,
// in dword s, the eight codes of k = 128 * block + 32 * s + 8 * (l / 16) + 0..7: what one 16x16x32 matrix instruction
// takes from that lane, so a wave's load of a block is one contiguous kilobyte and any group of 32, 64 or 128 ends
// with an instruction.  Inside a dword code 2i sits in nibble i and code 2i + 1 in nibble i + 4, 16 bits apart, so that one
// shift and one mask leave a pair of neighbouring codes in the two halves of a register.  Scales and zero points:
// [experts][column tiles][groups, up to a whole block][16 columns].  Columns past N and k past K hold zeros.
constexpr int kTileN = 16, kBlockK = 128;

struct W4Shape {
    int n_experts;
    int64_t N, K;
    int group;
    __host__ __device__ int64_t tiles() const { return (N + kTileN - 1) / kTileN; }
    __host__ __device__ int64_t blocks() const { return (K + kBlockK - 1) / kBlockK; }
    __host__ __device__ int64_t groups() const { return blocks() * (kBlockK / group); }
    bool ok() const {
        return n_experts > 0 && n_experts <= (1 << 20) && N > 0 && K > 0 && N <= (1 << 24) && K <= (1 << 24) &&
               (group == 32 || group == 64 || group == 128) && K % group == 0;
    }
};

__global__ __launch_bounds__(kBlock) void w4_pack_codes_kernel(const uint8_t *__restrict__ codes, W4Shape sh,
                                                               uint32_t *__restrict__ packed, int64_t total) {
    const int64_t step = (int64_t)gridDim.x * kBlock;
    for (int64_t d = (int64_t)blockIdx.x * kBlock + threadIdx.x; d < total; d += step) {
        const int s = (int)(d & 3), lane = (int)((d >> 2) & 63);
        int64_t rest = d >> 8;
        const int64_t block = rest % sh.blocks();
        rest /= sh.blocks();
        const int64_t tile = rest % sh.tiles(), e = rest / sh.tiles();
        const int64_t n = tile * kTileN + lane % 16, k0 = block * kBlockK + 32 * s + 8 * (lane / 16);
        uint32_t out = 0;
        if (n < sh.N && k0 < sh.K) {                         // K is a multiple of 32: all eight or none
            const uint8_t *c = codes + ((e * sh.N + n) * sh.K + k0) / 2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t b = c[i];
                out |= (b & 15u) << (4 * i);
                out |= (b >> 4) << (4 * i + 16);
            }
        }
        packed[d] = out;
    }
}

template <typename V>
__global__ __launch_bounds__(kBlock) void w4_pack_groups_kernel(const V *__restrict__ plane, W4Shape sh,
                                                                V *__restrict__ packed, int64_t total) {
    const int64_t step = (int64_t)gridDim.x * kBlock, groups = sh.K / sh.group;
    for (int64_t d = (int64_t)blockIdx.x * kBlock + threadIdx.x; d < total; d += step) {
        int64_t rest = d / kTileN;
        const int64_t g = rest % sh.groups();
        rest /= sh.groups();
        const int64_t n = rest % sh.tiles() * kTileN + d % kTileN, e = rest / sh.tiles();
        packed[d] = n < sh.N && g < groups ? plane[(e * sh.N + n) * groups + g] : V(0);
    }
}

size_t w4_packed_bytes(int n_experts, int64_t N, int64_t K, int group, int what) {
    const W4Shape sh{n_experts, N, K, group};
    if (!sh.ok()) return 0;
    const size_t cols = (size_t)n_experts * sh.tiles() * kTileN;
    if (what == 0) return cols * sh.blocks() * (kBlockK / 2);
    return cols * sh.groups() * (what == 1 ? 2 : 1);
}

int run_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int n_experts, int64_t N, int64_t K,
                int group, void *packed_codes, void *packed_scales, void *packed_zeros, hipStream_t s) {
    const W4Shape sh{n_experts, N, K, group};
    if (!sh.ok() || !codes || !scales || !packed_codes || !packed_scales || (zeros != nullptr) != (packed_zeros != nullptr) ||
        ((uintptr_t)packed_codes & 15) || (((uintptr_t)scales | (uintptr_t)packed_scales) & 1))
        return TERRACE_EINVAL;
    auto grid = [](int64_t n) {
        const int64_t b = (n + kBlock - 1) / kBlock;
        return (unsigned)(b < 65536 ? b : 65536);
    };
    const int64_t dwords = (int64_t)(w4_packed_bytes(n_experts, N, K, group, 0) / 4);
    const int64_t groups = (int64_t)w4_packed_bytes(n_experts, N, K, group, 2);
    w4_pack_codes_kernel<<<grid(dwords), kBlock, 0, s>>>(codes, sh, (uint32_t *)packed_codes, dwords);
    w4_pack_groups_kernel<uint16_t><<<grid(groups), kBlock, 0, s>>>((const uint16_t *)scales, sh, (uint16_t *)packed_scales,
                                                                    groups);
    if (zeros)
        w4_pack_groups_kernel<uint8_t><<<grid(groups), kBlock, 0, s>>>(zeros, sh, (uint8_t *)packed_zeros, groups);
    return check_launch();
}

// ---------------------------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------------------------
// A code c becomes the 16-bit float 16 + c by placing its four bits at the top of the mantissa of 16.0 (bf16: bits 3-6,
// f16: bits 6-9): two integer instructions for two codes.  The constant is taken out again after each group:
//   sum_k (c - z) x = sum_k (16 + c) x - (16 + z) * sum_k x,
// where sum_k x comes from one more matrix instruction per step against a column of ones, shared by all column tiles
// of the wave.  Both sums are fp32, so the constant costs 2-3 bits of 24, not of the inputs' 8 or 11.
template <int DT>
struct W4Type;
template <>
struct W4Type<TERRACE_BF16> {
    typedef bf16x8 Frag;
    static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u, kOnes = 0x3F803F80u;
    static __device__ __forceinline__ uint32_t place(uint32_t w, int i) {
        return i == 0 ? w << 3 : w >> (4 * i - 3);
    }
    static __device__ __forceinline__ f32x4 mfma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct W4Type<TERRACE_F16> {
    typedef f16x8 Frag;
    static constexpr uint32_t kMask = 0x03C003C0u, kBase = 0x4C004C00u, kOnes = 0x3C003C00u;
    static __device__ __forceinline__ uint32_t place(uint32_t w, int i) {
        return i < 2 ? w << (6 - 4 * i) : w >> (4 * i - 6);
    }
    static __device__ __forceinline__ f32x4 mfma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

template <int DT>
__device__ __forceinline__ typename W4Type<DT>::Frag w4_expand(uint32_t w) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (W4Type<DT>::place(w, i) & W4Type<DT>::kMask) | W4Type<DT>::kBase;
    return __builtin_bit_cast(typename W4Type<DT>::Frag, v);
}

// Which expert's rows a row tile holds.  Tiles of R rows are counted expert by expert; every wave finds its own by a scan
// over the counts, 64 lanes holding `per` consecutive experts each.  Counts are the caller's device data: each is taken
// into [0, P] and the sums saturate at P, so no count names a row outside the P rows.
struct RowTile {
    int expert;       // -1: past the last tile
    int first, rows;  // its rows
    int tiles, live;  // tiles and rows in all
};

__device__ __forceinline__ RowTile find_tile(const int64_t *__restrict__ counts, int n_experts, int P, int R, int tile) {
    const int lane = lane_id(), per = (n_experts + kWave - 1) / kWave, e0 = lane * per;
    int my_rows = 0, my_tiles = 0;
    for (int i = 0; i < per; ++i) {
        const int64_t c = e0 + i >= n_experts ? 0 : counts ? counts[e0 + i] : P;
        int n = c < 0 ? 0 : c > P ? P : (int)c;
        n = n < P - my_rows ? n : P - my_rows;
        my_rows += n;
        my_tiles += (n + R - 1) / R;
    }
    int rows = my_rows;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int r = __shfl_up(rows, d, kWave);
        if (lane >= d) rows = rows + r < P ? rows + r : P;
    }
    // a lane whose rows saturate keeps what is left for it; its tiles may then be fewer than it counted
    int before = __shfl_up(rows, 1, kWave);
    if (lane == 0) before = 0;
    if (rows - before < my_rows) {
        int left = rows - before;
        my_tiles = 0;
        for (int i = 0; i < per; ++i) {
            const int64_t c = e0 + i >= n_experts ? 0 : counts ? counts[e0 + i] : P;
            int n = c < 0 ? 0 : c > left ? left : (int)c;
            left -= n;
            my_tiles += (n + R - 1) / R;
        }
    }
    int upto = my_tiles;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int t = __shfl_up(upto, d, kWave);
        if (lane >= d) upto += t;
    }
    RowTile out;
    out.tiles = __shfl(upto, kWave - 1, kWave);
    out.live = __shfl(rows, kWave - 1, kWave);
    out.expert = -1;
    out.first = out.rows = 0;
    const uint64_t past = __ballot(upto > tile);
    if (past == 0) return out;
    // the owning lane walks its own experts
    if (lane == __builtin_ctzll(past)) {
        int t = upto - my_tiles, r = before;
        for (int i = 0; i < per; ++i) {
            const int64_t c = e0 + i >= n_experts ? 0 : counts ? counts[e0 + i] : P;
            const int n = c < 0 ? 0 : c > rows - r ? rows - r : (int)c;
            const int nt = (n + R - 1) / R;
            if (tile < t + nt) {
                const int skip = (tile - t) * R;
                out.expert = e0 + i;
                out.first = r + skip;
                out.rows = n - skip < R ? n - skip : R;
                break;
            }
            t += nt;
            r += n;
        }
    }
    const int owner = __builtin_ctzll(past);
    out.expert = read_lane(out.expert, owner);
    out.first = read_lane(out.first, owner);
    out.rows = read_lane(out.rows, owner);
    return out;
}

struct W4Args {
    const void *x;
    const int64_t *counts;
    int P;
    W4Shape sh;
    const u32x4 *codes;
    const uint16_t *scales;
    const uint8_t *zeros;      // NULL: 8
    int swiglu;
    int col_groups;            // workgroups along the columns
    void *out;
};

// A workgroup makes 32 columns -- two tiles: neighbours, or with `swiglu` the same columns of both halves -- of up to 16 * MT
// rows of one expert.  Its waves share out the blocks of k and are joined in LDS, in order.  GS: matrix steps per group.
constexpr int w4_max_waves(int mt) { return mt == 1 ? 8 : 4; }

template <int DT, int MT, int GS>
__global__ __launch_bounds__(w4_max_waves(MT) * kWave) void w4_linear_kernel(W4Args a) {
    typedef typename W4Type<DT>::Frag Frag;
    extern __shared__ float lds[];
    constexpr int R = 16 * MT;
    const int lane = lane_id(), w = wave_in_block(), waves = (int)(blockDim.x >> 6);
    const int cg = (int)(blockIdx.x % (unsigned)a.col_groups), tile = (int)(blockIdx.x / (unsigned)a.col_groups);
    const int grid_tiles = (int)(gridDim.x / (unsigned)a.col_groups);
    const int64_t N = a.sh.N, K = a.sh.K, out_cols = a.swiglu ? N / 2 : N;
    const RowTile rt = find_tile(a.counts, a.sh.n_experts, a.P, R, tile);
    const int c16 = lane & 15, q = lane >> 4;
    // the two columns of this lane
    const int64_t col0 = a.swiglu ? 16 * (int64_t)cg + c16 : 32 * (int64_t)cg + c16;
    const int64_t col1 = a.swiglu ? col0 + N / 2 : col0 + 16;
    uint16_t *out = (uint16_t *)a.out;
    if (rt.expert < 0) {                                     // rows no expert owns are zeros; the spare tiles write them
        for (int64_t r = rt.live + (tile - rt.tiles); r < a.P; r += grid_tiles - rt.tiles) {
            if (threadIdx.x < 16) {
                if (col0 < out_cols) out[r * out_cols + col0] = 0;
                if (!a.swiglu && col1 < out_cols) out[r * out_cols + col1] = 0;
            }
        }
        return;
    }
    const int64_t blocks = a.sh.blocks(), tiles = a.sh.tiles();
    const int64_t per = (blocks + waves - 1) / waves, b0 = w * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    const int64_t n0 = col0 < N ? col0 : N - 1, n1 = col1 < N ? col1 : N - 1;      // in bounds; dropped at the store
    const int64_t t0 = (int64_t)rt.expert * tiles + n0 / 16, t1 = (int64_t)rt.expert * tiles + n1 / 16;
    const u32x4 *w0 = a.codes + t0 * blocks * kWave + q * 16 + n0 % 16;
    const u32x4 *w1 = a.codes + t1 * blocks * kWave + q * 16 + n1 % 16;
    constexpr int GPB = 4 / GS;                              // groups per block
    const int64_t s0 = t0 * a.sh.groups() * kTileN + n0 % 16, s1 = t1 * a.sh.groups() * kTileN + n1 % 16;
    const uint16_t *xr[MT];
    bool has[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        has[m] = 16 * m + c16 < rt.rows;
        xr[m] = (const uint16_t *)a.x + (int64_t)(rt.first + (has[m] ? 16 * m + c16 : 0)) * K + 8 * q;
    }
    const u32x4 ones4 = {W4Type<DT>::kOnes, W4Type<DT>::kOnes, W4Type<DT>::kOnes, W4Type<DT>::kOnes};
    const Frag ones = __builtin_bit_cast(Frag, ones4);
    f32x4 total[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) total[m][0] = total[m][1] = f32x4{0, 0, 0, 0};

    struct Block {
        u32x4 w[2];
        u32x4 x[MT][4];
        uint16_t s[2][GPB];
        uint8_t z[2][GPB];
    };
    auto fetch = [&](int64_t b, Block &k) {
        k.w[0] = w0[b * kWave];
        k.w[1] = w1[b * kWave];
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
            k.s[0][g] = a.scales[s0 + (b * GPB + g) * kTileN];
            k.s[1][g] = a.scales[s1 + (b * GPB + g) * kTileN];
            k.z[0][g] = k.z[1][g] = 8;
            if (a.zeros) {
                k.z[0][g] = a.zeros[s0 + (b * GPB + g) * kTileN];
                k.z[1][g] = a.zeros[s1 + (b * GPB + g) * kTileN];
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t at = b * kBlockK + 32 * s;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                k.x[m][s] = zero_of<u32x4>();
                if (has[m] && at < K) k.x[m][s] = *(const u32x4 *)(xr[m] + at);
            }
        }
    };
    auto use = [&](const Block &k) {
        f32x4 acc[MT][2], sum[MT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const Frag f0 = w4_expand<DT>(k.w[0][s]), f1 = w4_expand<DT>(k.w[1][s]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const Frag x = __builtin_bit_cast(Frag, k.x[m][s]);
                const f32x4 zero = {0, 0, 0, 0};
                const bool first = s % GS == 0;
                acc[m][0] = W4Type<DT>::mfma(x, f0, first ? zero : acc[m][0]);
                acc[m][1] = W4Type<DT>::mfma(x, f1, first ? zero : acc[m][1]);
                sum[m] = W4Type<DT>::mfma(x, ones, first ? zero : sum[m]);
            }
            if (s % GS == GS - 1) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float scale;
                    const uint16_t bits = k.s[t][s / GS];
                    if constexpr (DT == TERRACE_BF16) scale = bf16_bits_to_f32(bits);
                    else scale = __half2float(__ushort_as_half(bits));
                    const float off = -(16.0f + (float)k.z[t][s / GS]);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            total[m][t][i] = __fmaf_rn(scale, __fmaf_rn(off, sum[m][i], acc[m][t][i]), total[m][t][i]);
                }
            }
        }
    };
    if (b0 < b1) {
        Block cur, next;
        fetch(b0, cur);
        for (int64_t b = b0; b < b1; ++b) {
            if (b + 1 < b1) fetch(b + 1, next);
            use(cur);
            cur = next;
        }
    }
    // join the waves: lds[w][m][t][i][lane]
    constexpr int kPer = MT * 2 * 4;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) lds[((w * MT + m) * 8 + t * 4 + i) * kWave + lane] = total[m][t][i];
    __syncthreads();
    for (int j = w; j < MT * 4; j += waves) {                // row (m, i) of each lane's quarter, both columns
        const int m = j >> 2, i = j & 3;
        float v[2] = {0.0f, 0.0f};
        for (int x = 0; x < waves; ++x) {
            v[0] += lds[(x * kPer + m * 8 + i) * kWave + lane];
            v[1] += lds[(x * kPer + m * 8 + 4 + i) * kWave + lane];
        }
        const int row = 16 * m + 4 * q + i;
        if (row >= rt.rows) continue;
        uint16_t *o = out + (int64_t)(rt.first + row) * out_cols;
        if (a.swiglu) {
            const float y = v[0] / (1.0f + __expf(-v[0])) * v[1];
            if (col0 < out_cols) o[col0] = (uint16_t)to_bits16<DT>(y);
        } else {
            if (col0 < out_cols) o[col0] = (uint16_t)to_bits16<DT>(v[0]);
            if (col1 < out_cols) o[col1] = (uint16_t)to_bits16<DT>(v[1]);
        }
    }
}

template <int DT, int MT>
static void launch_w4_g(const W4Args &a, unsigned grid, int waves, hipStream_t s) {
    const size_t lds = (size_t)waves * MT * 8 * kWave * sizeof(float);
    if (a.sh.group == 128) w4_linear_kernel<DT, MT, 4><<<grid, waves * kWave, lds, s>>>(a);
    else if (a.sh.group == 64) w4_linear_kernel<DT, MT, 2><<<grid, waves * kWave, lds, s>>>(a);
    else w4_linear_kernel<DT, MT, 1><<<grid, waves * kWave, lds, s>>>(a);
}

int run_w4_linear(const void *x, int dtype, int64_t P, const int64_t *counts, const void *codes, const void *scales,
                  const void *zeros, int n_experts, int64_t N, int64_t K, int group, int swiglu, void *out,
                  hipStream_t s) {
    const W4Shape sh{n_experts, N, K, group};
    if (P < 0 || P > ((int64_t)1 << 30) || (dtype != TERRACE_BF16 && dtype != TERRACE_F16) || !sh.ok() || (swiglu && N % 2))
        return TERRACE_EINVAL;
    if (P == 0) return TERRACE_OK;
    if (!x || (!counts && n_experts != 1) || !codes || !scales || !out || (((uintptr_t)x | (uintptr_t)codes) & 15) ||
        (((uintptr_t)scales | (uintptr_t)out) & 1))
        return TERRACE_EINVAL;
    const int64_t busy = P < n_experts ? P : n_experts;      // experts that can hold a row
    const int64_t mean = (P + busy - 1) / busy;
    const int mt = mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
    const int R = 16 * mt;
    const int64_t col_groups = swiglu ? (N / 2 + 15) / 16 : (N + 31) / 32;
    const int64_t row_tiles = busy + (P - busy) / R + 1;     // the most there can be, and one for rows without expert
    if (col_groups * row_tiles >= (int64_t)1 << 23) return TERRACE_EINVAL;   // 512 threads each: HIP's grid limit
    int waves = 4;
    if (mt == 1 && col_groups * (row_tiles - 1) * waves < 4096 && sh.blocks() > waves) waves = 8;
    const W4Args a{x, counts, (int)P, sh, (const u32x4 *)codes, (const uint16_t *)scales, (const uint8_t *)zeros, swiglu,
                   (int)col_groups, out};
    const unsigned grid = (unsigned)(col_groups * row_tiles);
#define TERRACE_W4(DT)                                  \
    if (mt == 1) launch_w4_g<DT, 1>(a, grid, waves, s); \
    else if (mt == 2) launch_w4_g<DT, 2>(a, grid, waves, s); \
    else launch_w4_g<DT, 4>(a, grid, waves, s)
    if (dtype == TERRACE_BF16) { TERRACE_W4(TERRACE_BF16); }
    else { TERRACE_W4(TERRACE_F16); }
#undef TERRACE_W4
    return check_launch();
}

}  // namespace terrace
