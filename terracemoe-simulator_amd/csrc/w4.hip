// The experts' products for a few rows each, on 4-bit weights with group scales.
//
//   w4_pack_*_kernel                codes, scales and zero points into the order the product reads them (once per weight)
//   w4_few_kernel, w4_many_kernel   out[i, n] = sum_k scale[e, n, k / g] * (code[e, n, k] - zero[e, n, k / g]) * x[i, k]
//                     for the rows i of expert e; optionally silu(first half of the columns) * (second half)
//
// Few rows per expert, so the product reads every code once and does little with it: it is bound by the HBM bytes of
// the weights of the experts that hold a row.  What the matrix cores are used for here is not their rate but that one
// instruction multiplies 8 codes of a lane with up to 16 rows.
#include "common.hpp"

namespace terrace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------------------------
// codes as 16-bit floats
// ---------------------------------------------------------------------------------------------
// A code c becomes the 16-bit float 16 + c by placing its four bits at the top of the mantissa of 16.0 (bf16: bits 3-6,
// f16: bits 6-9): one turn and one and-or for two codes.  The constant is taken out again group by group,
//   sum_k (c - z) x = sum_k (16 + c) x - (16 + z) * sum_k x,
// the second sum by matrix instructions too (w4_use).  Everything is added in fp32, so the constant costs 2-3 bits of
// 24, not of the inputs' 8 or 11.  An infinite x, or a bf16 x whose multiples pass 2^128, makes both sums infinite where
// their difference need not be: a result that is not finite is taken again from the definition (w4_plain).
template <int DT>
struct W4Type;
template <>
struct W4Type<TERRACE_BF16> {
    typedef bf16x8 Frag;
    static constexpr int kShift = 3;
    static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u, kOnes = 0x3F803F80u, kLess24 = 0xC1C0C1C0u;
    static __device__ __forceinline__ f32x4 mfma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct W4Type<TERRACE_F16> {
    typedef f16x8 Frag;
    static constexpr int kShift = 6;
    static constexpr uint32_t kMask = 0x03C003C0u, kBase = 0x4C004C00u, kOnes = 0x3C003C00u, kLess24 = 0xCE00CE00u;
    static __device__ __forceinline__ f32x4 mfma(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

template <int DT>
__device__ __forceinline__ typename W4Type<DT>::Frag w4_frag(uint32_t pair) {
    const u32x4 v = {pair, pair, pair, pair};
    return __builtin_bit_cast(typename W4Type<DT>::Frag, v);
}
// `base`: W4Type::kBase in a vector register (one and-or takes only one constant from elsewhere)
template <int DT>
__device__ __forceinline__ typename W4Type<DT>::Frag w4_expand(uint32_t w, uint32_t base) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = i == 0 ? w : __builtin_amdgcn_alignbit(w, w, 4 * i);
        v[i] = (t & W4Type<DT>::kMask) | base;
    }
    return __builtin_bit_cast(typename W4Type<DT>::Frag, v);
}

// ---------------------------------------------------------------------------------------------
// packed layout
// ---------------------------------------------------------------------------------------------
// Codes: [experts][column tiles of 16][blocks of 128 k][64 lanes][4 dwords].  Lane l holds column l % 16 of its tile and,
// in dword s, the eight codes of k = 128 * block + 32 * s + 8 * (l / 16) + 0..7: what one 16x16x32 matrix instruction
// takes from that lane, so a wave's load of a block is one contiguous kilobyte and any group of 32, 64 or 128 ends
// with an instruction.  Inside a dword code 2i sits in nibble i and code 2i + 1 in nibble i + 4, 16 bits apart, and the
// whole is turned left by the place a code takes in its 16-bit float (below): turning right by 4i puts a pair of
// neighbouring codes where the two halves of a register want them.  Scales and zero points:
// [experts][column tiles][blocks][16 columns][groups of a block], so a lane has those of a block in one load.  Columns
// past N and k past K hold zeros.
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
               (group == 32 || group == 64 || group == 128) && K % group == 0 &&
               tiles() * blocks() < (1 << 21);               // an expert's codes stay below 2^31 bytes: 32-bit offsets
    }
};

__global__ __launch_bounds__(kBlock) void w4_pack_codes_kernel(const uint8_t *__restrict__ codes, W4Shape sh,
                                                               int turn, uint32_t *__restrict__ packed, int64_t total) {
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
        packed[d] = out << turn | out >> (32 - turn);
    }
}

template <typename V>
__global__ __launch_bounds__(kBlock) void w4_pack_groups_kernel(const V *__restrict__ plane, W4Shape sh,
                                                                V *__restrict__ packed, int64_t total) {
    const int64_t step = (int64_t)gridDim.x * kBlock, groups = sh.K / sh.group;
    for (int64_t d = (int64_t)blockIdx.x * kBlock + threadIdx.x; d < total; d += step) {
        const int gpb = kBlockK / sh.group;
        int64_t rest = d / gpb;
        const int64_t col = rest % kTileN;
        rest /= kTileN;
        const int64_t g = rest % sh.blocks() * gpb + d % gpb;
        rest /= sh.blocks();
        const int64_t n = rest % sh.tiles() * kTileN + col, e = rest / sh.tiles();
        V v = n < sh.N && g < groups ? plane[(e * sh.N + n) * groups + g] : V(0);
        if (sizeof(V) == 1) v &= 15;                         // a zero point has four bits: more would reach the exponent
        packed[d] = v;
    }
}

size_t w4_packed_bytes(int n_experts, int64_t N, int64_t K, int group, int what) {
    const W4Shape sh{n_experts, N, K, group};
    if (!sh.ok()) return 0;
    const size_t cols = (size_t)n_experts * sh.tiles() * kTileN;
    if (what == 0) return cols * sh.blocks() * (kBlockK / 2);
    return cols * sh.groups() * (what == 1 ? 2 : 1);
}

int run_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int dtype, int n_experts, int64_t N,
                int64_t K, int group, void *packed_codes, void *packed_scales, void *packed_zeros, hipStream_t s) {
    const W4Shape sh{n_experts, N, K, group};
    if (!sh.ok() || (dtype != TERRACE_BF16 && dtype != TERRACE_F16) || !codes || !scales || !packed_codes || !packed_scales || (zeros != nullptr) != (packed_zeros != nullptr) ||
        ((uintptr_t)packed_codes & 15) || (((uintptr_t)scales | (uintptr_t)packed_scales) & 1))
        return TERRACE_EINVAL;
    auto grid = [](int64_t n) {
        const int64_t b = (n + kBlock - 1) / kBlock;
        return (unsigned)(b < 65536 ? b : 65536);
    };
    const int64_t dwords = (int64_t)(w4_packed_bytes(n_experts, N, K, group, 0) / 4);
    const int64_t groups = (int64_t)w4_packed_bytes(n_experts, N, K, group, 2);
    w4_pack_codes_kernel<<<grid(dwords), kBlock, 0, s>>>(
        codes, sh, dtype == TERRACE_BF16 ? W4Type<TERRACE_BF16>::kShift : W4Type<TERRACE_F16>::kShift,
        (uint32_t *)packed_codes, dwords);
    w4_pack_groups_kernel<uint16_t><<<grid(groups), kBlock, 0, s>>>((const uint16_t *)scales, sh, (uint16_t *)packed_scales,
                                                                    groups);
    if (zeros)
        w4_pack_groups_kernel<uint8_t><<<grid(groups), kBlock, 0, s>>>(zeros, sh, (uint8_t *)packed_zeros, groups);
    return check_launch();
}

// ---------------------------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------------------------
// Which expert's rows a row tile holds.  Tiles of R rows are counted expert by expert; every wave finds its own by scans
// over the counts, a lane an expert, 64 at a time.  Counts are the caller's device data: each is taken into [0, P] and the
// sums saturate at P, so no count names a row outside the P rows.
struct RowTile {
    int expert;       // -1: past the last tile
    int first, rows;  // its rows
    int tiles, live;  // past the last tile only: tiles and rows in all
};

// Inclusive scan over the wave, every sum cut at `most` (all values in [0, most], most <= 2^30).
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v, int most) {
    const int t = v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
    return t < most ? t : most;
}
__device__ __forceinline__ int wave_scan(int v, int most) {
    v = scan_step<0x111, 0xF>(v, most);                      // row_shr:1, 2, 4, 8 inside the rows of 16 lanes
    v = scan_step<0x112, 0xF>(v, most);
    v = scan_step<0x114, 0xF>(v, most);
    v = scan_step<0x118, 0xF>(v, most);
    v = scan_step<0x142, 0xA>(v, most);                      // and the rows' totals upwards
    return scan_step<0x143, 0xC>(v, most);
}

__device__ __forceinline__ RowTile find_tile(const int64_t *__restrict__ counts, int n_experts, int P, int R, int tile) {
    const int lane = lane_id();
    int rows = 0, tiles = 0;                                 // before the experts looked at
    constexpr int kLoads = 4;                                // 256 experts' counts in flight at once
    for (int e0 = 0; e0 < n_experts; e0 += kLoads * kWave) {
        int64_t c[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int e = e0 + j * kWave + lane;
            c[j] = e >= n_experts ? 0 : counts ? counts[e] : P;
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int n = c[j] < 0 ? 0 : c[j] > P ? P : (int)c[j];
            int upto = wave_scan(n, P) + rows;
            if (upto > P) upto = P;
            int from = __shfl_up(upto, 1, kWave);
            if (lane == 0) from = rows;
            const int mine = (upto - from + R - 1) / R;
            const int upto_tiles = wave_scan(mine, P) + tiles;
            const uint64_t past = __ballot(upto_tiles > tile);
            if (past) {
                const int at = __builtin_ctzll(past);
                const int skip = (tile - read_lane(upto_tiles - mine, at)) * R;
                const int first = read_lane(from, at), n_rows = read_lane(upto, at) - first - skip;
                return {e0 + j * kWave + at, first + skip, n_rows < R ? n_rows : R, 0, 0};
            }
            rows = read_lane(upto, kWave - 1);
            tiles = read_lane(upto_tiles, kWave - 1);
        }
    }
    return {-1, 0, 0, tiles, rows};
}

struct W4Args {
    const void *x;
    const int64_t *counts;     // NULL: one expert with all rows
    int P;
    W4Shape sh;
    const u32x4 *codes;
    const uint16_t *scales;
    const uint8_t *zeros;      // NULL: 8
    int swiglu;
    void *out;
    // worked out once on the host
    int out_cols;
    int tiles, blocks;         // column tiles of the weights and packed blocks of k
    int full, rest;            // whole blocks of k, and the steps of 32 in what is left
    int col_blocks;            // workgroups along the columns
    int split, per;            // few rows: waves that share out the k of one set of columns, and the whole blocks of each
    int sets;                  // few rows: sets of columns in a workgroup
};

// Rows no expert owns are zeros; the workgroups past the last tile write the columns [lo, hi) of them.
__device__ __forceinline__ void w4_zero_rows(const W4Args &a, const RowTile &rt, int tile, int lo, int hi) {
    const int spare = (int)(gridDim.x / (unsigned)a.col_blocks) - rt.tiles;
    if (hi > a.out_cols) hi = a.out_cols;
    for (int64_t r = rt.live + (tile - rt.tiles); r < a.P; r += spare)
        for (int c = lo + (int)threadIdx.x; c < hi; c += (int)blockDim.x) ((uint16_t *)a.out)[r * a.out_cols + c] = 0;
}

// A lane's column of one expert: byte offsets of its codes and (in groups) of its scales from the expert's first.
struct W4Expert {
    const uint8_t *codes, *scales, *zeros;                   // of the tile's expert; zeros may be NULL
};
struct W4Column {
    uint32_t codes, groups;
};
__device__ __forceinline__ W4Expert w4_expert(const W4Args &a, int expert, int gpb) {
    const int64_t blocks = (int64_t)expert * a.tiles * a.blocks, groups = blocks * (gpb * kTileN);
    return {(const uint8_t *)a.codes + blocks * 1024, (const uint8_t *)a.scales + 2 * groups,
            a.zeros ? a.zeros + groups : nullptr};
}
__device__ __forceinline__ W4Column w4_column(const W4Args &a, int col, int q, int gpb) {
    const uint32_t n = (uint32_t)(col < (int)a.sh.N ? col : (int)a.sh.N - 1);      // in bounds; dropped at the store
    const uint32_t block = n / kTileN * (uint32_t)a.blocks;
    return {block * 1024u + (uint32_t)(q * 16 + n % kTileN) * 16u, (block * kTileN + n % kTileN) * gpb};
}

// T tiles of a block of k: codes, scales and zero points of this lane's columns.
template <int GPB>
struct GroupBits;
template <>
struct GroupBits<1> { typedef uint16_t S; typedef uint8_t Z; };
template <>
struct GroupBits<2> { typedef uint32_t S; typedef uint16_t Z; };
template <>
struct GroupBits<4> { typedef u32x2 S; typedef uint32_t Z; };
template <int T, int GPB, bool ZEROS>
struct W4Block {
    u32x4 w[T];
    static constexpr int kWords = GPB == 4 ? 2 : 1;
    uint32_t s[T][kWords];                                   // a scale in each half
    uint32_t z[ZEROS ? T : 1];                               // a zero point in each byte
    template <bool STREAM>
    __device__ __forceinline__ void fetch(const W4Expert &e, const W4Column *col, int b) {
        const uint8_t *codes = e.codes + (int64_t)b * 1024, *scales = e.scales + (int64_t)b * (2 * GPB * kTileN);
        const uint8_t *zeros = ZEROS ? e.zeros + (int64_t)b * (GPB * kTileN) : nullptr;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            // a scalar base and a 32-bit offset: the offsets are kept apart, or the compiler adds them up ahead of the
            // loop and pays a 64-bit vector add a load
            uint32_t at = col[t].codes, group = col[t].groups;
            asm volatile("" : "+v"(at), "+v"(group));
            w[t] = STREAM ? ld_stream((const u32x4 *)(codes + at)) : *(const u32x4 *)(codes + at);
            const auto v = *(const typename GroupBits<GPB>::S *)(scales + 2u * group);
            if constexpr (GPB == 4) {
                s[t][0] = v[0];
                s[t][1] = v[1];
            } else {
                s[t][0] = v;
            }
            if constexpr (ZEROS) z[t] = *(const typename GroupBits<GPB>::Z *)(zeros + group);
        }
    }
};

// total += the block's products: x(m, s) gives the rows' fragment of step s.  What takes the constant out:
//   no zero points       sum_k -24 x, summed first by matrix instructions, is where every tile's sum of a group starts
//   ZEROS, one row tile  a matrix instruction more per tile and step, against -(16 + z)
//   ZEROS, more          sum_k x by matrix instructions, once for all tiles, and a multiply-add per result
template <int DT, int MT, int T, int GS, bool ZEROS, typename X>
__device__ __forceinline__ void w4_use(W4Block<T, 4 / GS, ZEROS> &k, X x, f32x4 (*total)[T]) {
    typedef W4Type<DT> Type;
    typedef typename Type::Frag Frag;
    uint32_t base = Type::kBase;
    asm volatile("" : "+v"(base));
    // what was fetched stays as it came until here: without this the compiler unpacks it where it arrives, and a ring of
    // unpacked blocks does not fit the registers
#pragma unroll
    for (int t = 0; t < T; ++t) {
        asm volatile("" : "+v"(k.w[t]));
        if constexpr (ZEROS) asm volatile("" : "+v"(k.z[t]));
#pragma unroll
        for (int i = 0; i < W4Block<T, 4 / GS, ZEROS>::kWords; ++i) asm volatile("" : "+v"(k.s[t][i]));
    }
    constexpr bool kSum = ZEROS && MT > 1, kTile = ZEROS && MT == 1;
#pragma unroll
    for (int g = 0; g < 4 / GS; ++g) {
        f32x4 acc[MT][T], sum[MT];
        const f32x4 zero = {0, 0, 0, 0};
        if constexpr (!kTile) {
            const Frag c = w4_frag<DT>(kSum ? Type::kOnes : Type::kLess24);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                sum[m] = zero;
#pragma unroll
                for (int s = 0; s < GS; ++s) sum[m] = Type::mfma(__builtin_bit_cast(Frag, x(m, g * GS + s)), c, sum[m]);
            }
        }
        Frag less[T];
        if constexpr (kTile) {
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const uint32_t z = (k.z[t] >> (8 * g)) & 0xFFu, half = 0x8000u | (Type::kBase & 0x7FFFu) | (z << Type::kShift);
                less[t] = w4_frag<DT>(half | half << 16);
            }
        }
#pragma unroll
        for (int s = 0; s < GS; ++s) {
            Frag xs[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) xs[m] = __builtin_bit_cast(Frag, x(m, g * GS + s));
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const Frag f = w4_expand<DT>(k.w[t][g * GS + s], base);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const f32x4 from = s ? acc[m][t] : ZEROS ? zero : sum[m];
                    acc[m][t] = Type::mfma(xs[m], f, from);
                    if constexpr (kTile) acc[m][t] = Type::mfma(xs[m], less[t], acc[m][t]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);               // one step's expanded codes at a time in registers
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float scale;
            const uint32_t word = k.s[t][g / 2];
            if constexpr (DT == TERRACE_BF16) scale = g & 1 ? __uint_as_float(word & 0xFFFF0000u) : __uint_as_float(word << 16);
            else scale = __half2float(__ushort_as_half((unsigned short)(g & 1 ? word >> 16 : word)));
            float off = 0.0f;
            if constexpr (kSum) off = -16.0f - (float)((k.z[t] >> (8 * g)) & 0xFFu);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = acc[m][t][i];
                    if constexpr (kSum) v = __fmaf_rn(off, sum[m][i], v);
                    total[m][t][i] = __fmaf_rn(scale, v, total[m][t][i]);
                }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

__device__ __forceinline__ bool w4_finite(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// One result from the definition, sum_k (scale * (code - zero)) * x[k] over k in order, by one lane: an infinite x gives
// an infinity, or NaN where its weight is 0, and a finite sum is found although (16 + code) x left the range.  Reached by
// results that are not finite only; what waits in it is one lane's chain of loads.  One token through the gate and up
// projections of 8 experts (4096 x 7168): 27 us, 420-480 with an infinity in one row, 750-780 with one in all eight; 2048 rows
// over 64 experts of 4096 x 4096: 155 us, 1.0-1.1 ms with one such row, 13.5-14.5 ms with nothing else.  NaN ends the sum: with
// one at the start of every row 32 and 179 us.
template <int DT, int GS, bool ZEROS>
__device__ __forceinline__ float w4_plain(const W4Args &a, const W4Expert &e, int col, const uint8_t *row) {
    constexpr int kGpb = 4 / GS;
    float sum = 0.0f;
#pragma unroll 1
    for (int k = 0; k < (int)a.sh.K; k += 8) {               // one dword of codes; K is a multiple of 32
        const int block = k / kBlockK, step = k / 32 % 4;
        const W4Column c = w4_column(a, col, k / 8 % 4, kGpb);
        const uint32_t w = *(const uint32_t *)(e.codes + (int64_t)block * 1024 + c.codes + 4 * step);
        const uint32_t codes = __builtin_amdgcn_alignbit(w, w, W4Type<DT>::kShift);          // as before the turn of the packing
        const int64_t group = (int64_t)block * (kGpb * kTileN) + c.groups + step / GS;
        const uint32_t s = ((const uint16_t *)e.scales)[group];
        float scale;
        if constexpr (DT == TERRACE_BF16) scale = bf16_bits_to_f32(s);
        else scale = __half2float(__ushort_as_half((unsigned short)s));
        const int zero = ZEROS ? (int)e.zeros[group] : 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int code = (int)(codes >> (4 * (i / 2) + 16 * (i & 1))) & 15;
            float x;
            load_floats<DT, 1>(row, k + i, &x);
            sum = __fmaf_rn(scale * (float)(code - zero), x, sum);
        }
        if (sum != sum) break;                               // NaN stays
    }
    return sum;
}

__device__ __forceinline__ float w4_swiglu(float gate, float up) { return gate / (1.0f + __expf(-gate)) * up; }

// Few rows: tiles of 16.  One token through the gate and up projections of 8 experts (121 MB) 25 us, 4.8 TB/s; 512 rows
// over 174 busy experts of 7168 x 2048 (1.33 GB) 245 us, 5.4 TB/s, with vector instructions in 45 % of the cycles.  A set of
// 32 columns -- two tiles: neighbours, or with `swiglu` the same columns of both halves -- is the work of `split` waves that share out the blocks of k and are joined in LDS, in order; a workgroup holds 4 or 8
// waves and so 4 / split or 8 / split sets.  The rows' fragments come straight from memory (a few rows: L1 and L2), and
// codes and rows are fetched kAhead blocks ahead, because the codes come from HBM and nothing else hides their latency.
// (One token, measured before the codes were loaded around the cache: 27.8 us with two blocks ahead, 31.1 with four, whose
// registers cost waves; k shared out among up to 8192 waves and not 4096 30.4 us for 27.8, one token's down projection
// 22.3 for 17.2.)
constexpr int kAhead = 2;
constexpr int kMaxSplit = 8;

template <int DT, int GS, bool ZEROS>
__global__ __launch_bounds__(kMaxSplit * kWave) void w4_few_kernel(W4Args a) {
    __shared__ float lds[kMaxSplit][8][kWave];
    const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_in_block());
    const int cb = (int)(blockIdx.x % (unsigned)a.col_blocks), tile = (int)(blockIdx.x / (unsigned)a.col_blocks);
    const int width = a.swiglu ? 16 : 32, lo = cb * a.sets * width;
    const RowTile rt = find_tile(a.counts, a.sh.n_experts, a.P, 16, tile);
    if (rt.expert < 0) {
        w4_zero_rows(a, rt, tile, lo, lo + a.sets * width);
        return;
    }
    const int c16 = lane & 15, q = lane >> 4, set = w / a.split, part = w - set * a.split;
    const int col0 = lo + set * width + c16, col1 = a.swiglu ? col0 + a.out_cols : col0 + 16;
    const W4Expert we = w4_expert(a, rt.expert, 4 / GS);
    const W4Column col[2] = {w4_column(a, col0, q, 4 / GS), w4_column(a, col1, q, 4 / GS)};
    const int b0 = part * a.per < a.full ? part * a.per : a.full, b1 = b0 + a.per < a.full ? b0 + a.per : a.full;
    // a lane without a row reads the tile's first one: the same lines, and its results are dropped
    const uint8_t *xt = (const uint8_t *)a.x + (int64_t)rt.first * a.sh.K * 2;
    const uint32_t xo = (uint32_t)((c16 < rt.rows ? c16 : 0) * (int)a.sh.K + 8 * q) * 2u;
    f32x4 total[1][2] = {{f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}};
    struct Block {
        W4Block<2, 4 / GS, ZEROS> k;
        u32x4 x[4];
    };
    auto fetch = [&](int b, Block &f) {
        f.k.template fetch<true>(we, col, b);
        const uint8_t *xb = xt + (int64_t)b * (2 * kBlockK);
        uint32_t o = xo;
        asm volatile("" : "+v"(o));
#pragma unroll
        for (int s = 0; s < 4; ++s) f.x[s] = *(const u32x4 *)(xb + o + 64 * s);
    };
    auto use = [&](Block &f) {
        w4_use<DT, 1, 2, GS, ZEROS>(f.k, [&](int, int s) { return f.x[s]; }, total);
    };
    if (b0 < b1) {
        Block ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) fetch(b0 + i < b1 ? b0 + i : b1 - 1, ring[i]);
        int b = b0;
        for (; b + kAhead <= b1; b += kAhead) {              // past the end the last block is fetched again, from cache
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                use(ring[i]);
                fetch(b + kAhead + i < b1 ? b + kAhead + i : b1 - 1, ring[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) {
            if (b + i < b1) use(ring[i]);
        }
    }
    if (a.rest && part == a.split - 1) {                     // a K that is no multiple of 128: zeros past it
        Block f;
        f.k.template fetch<true>(we, col, a.full);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            f.x[s] = zero_of<u32x4>();
            if (s < a.rest) f.x[s] = *(const u32x4 *)(xt + (int64_t)a.full * (2 * kBlockK) + xo + 64 * s);
        }
        use(f);
    }
    uint32_t again = 0;                                      // rows of this lane's quarter with a sum that is not finite
    auto store = [&](int i, float v0, float v1) {            // row i of this lane's quarter
        const int row = 4 * q + i;
        if (row >= rt.rows) return;
        if (!w4_finite(v0) || !w4_finite(v1)) again |= 1u << i;
        uint16_t *o = (uint16_t *)a.out + (int64_t)(rt.first + row) * a.out_cols;
        if (a.swiglu) {
            if (col0 < a.out_cols) o[col0] = (uint16_t)to_bits16<DT>(w4_swiglu(v0, v1));
        } else {
            if (col0 < a.out_cols) o[col0] = (uint16_t)to_bits16<DT>(v0);
            if (col1 < a.out_cols) o[col1] = (uint16_t)to_bits16<DT>(v1);
        }
    };
    if (a.split == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store(i, total[0][0][i], total[0][1][i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lds[w][i][lane] = total[0][0][i];
            lds[w][4 + i][lane] = total[0][1][i];
        }
        __syncthreads();
        for (int i = part; i < 4; i += a.split) {
            float v0 = 0.0f, v1 = 0.0f;
            for (int y = w - part; y < w - part + a.split; ++y) {
                v0 += lds[y][i][lane];
                v1 += lds[y][4 + i][lane];
            }
            store(i, v0, v1);
        }
    }
    for (uint32_t left = again; left; left &= left - 1) {
        const int i = __builtin_ctz(left);
        const uint8_t *row = xt + (int64_t)(4 * q + i) * a.sh.K * 2;
        float v[2];
#pragma unroll 1
        for (int j = 0; j < 2; ++j) {
            const float r = w4_plain<DT, GS, ZEROS>(a, we, j ? col1 : col0, row);
            v[0] = j ? v[0] : r;
            v[1] = r;
        }
        store(i, v[0], v[1]);
    }
}

// Tens of rows: tiles of 16 * MT.  A workgroup of four waves makes 256 columns, each wave four tiles (with `swiglu` two of
// each half), so the rows of a block of k are read once for 256 columns: they go through LDS in the order the matrix
// instructions take them, while every wave streams its own codes two blocks ahead.  2048 rows over 64 experts of 4096 x
// 4096 199-211 us (0.33 PFLOP/s, 612 MB), 256 rows of each of 8 experts 85-90 us.  By counters vector instructions (307 a block
// and wave, and the issue of 40 matrix instructions) fill 60 % of the cycles and matrix instructions 28 %: neither is full, and two
// waves a SIMD do not hide one behind the other.
//
// Against the kernel above (few / tiled, us, without and with zero points): 64 experts of 2048 x 7168, 4 rows each 94 / 99
// and 100 / 114, 8 rows 105 / 100 and 112 / 114, 16 rows 135 / 102 and 141 / 117; of 4096 x 4096 8 rows 116 / 129 and 123 / 138,
// 12 rows 133 / 132 and 143 / 138, 16 rows 150 / 134 and 157 / 139; 256 experts of 7168 x 2048, 8 rows 447 / 399 and
// 465 / 475.  So it is taken from more than 8 rows a busy expert on, and where its grid holds a workgroup for every CU:
// with half of them, 8 experts of 4096 x 4096, 16 rows 27 / 34 and 27 / 41 and 32 rows 42 / 35 and 45 / 42; with an eighth to a
// quarter, one matrix of 7168 x 7168 at 64 rows 37 / 87, of 16384 x 4096 43 / 54.
//
// MT 4 reads and expands the codes once for 64 rows, at up to 250 registers; with zero points it does not fit them.  32 / 64
// rows a tile: 8 experts of 4096 x 4096, groups of 64, 64 rows each 37 / 73 us, 128 rows 54 / 58, 256 rows 96 / 87; 32 experts of
// 2048 x 7168, 64 rows 91 / 94, 128 rows 173 / 153, 256 rows 327 / 299.  With zero points 64 rows 99 / 194, 128 rows 193 / 245,
// 256 rows 384 / 495 (spilling): not built.
constexpr int kManyTiles = 4;
// (two waves a SIMD at least: with a whole SIMD's registers to itself the compiler puts the sums into accumulation
// registers and copies each out again before the multiply-add, a fifth of the kernel's instructions)
template <int DT, int MT, int GS, bool ZEROS>
__global__ __launch_bounds__(4 * kWave, 2) void w4_many_kernel(W4Args a) {
    constexpr int R = 16 * MT, T = kManyTiles;
    __shared__ u32x4 rows[2][4][MT][kWave];                  // [buffer][step][16 rows][lane]
    const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_in_block());
    const int cb = (int)(blockIdx.x % (unsigned)a.col_blocks), tile = (int)(blockIdx.x / (unsigned)a.col_blocks);
    const int width = a.swiglu ? T * 8 : T * 16, lo = cb * 4 * width;
    const RowTile rt = find_tile(a.counts, a.sh.n_experts, a.P, R, tile);
    if (rt.expert < 0) {
        w4_zero_rows(a, rt, tile, lo, lo + 4 * width);
        return;
    }
    const int c16 = lane & 15, q = lane >> 4;
    const W4Expert we = w4_expert(a, rt.expert, 4 / GS);
    // swiglu: tiles 0 and 2 of the first half, 1 and 3 their partners
    auto column = [&](int t) { return lo + w * width + (a.swiglu ? (t >> 1) * 16 + (t & 1) * a.out_cols : t * 16); };
    W4Column col[T];
#pragma unroll
    for (int t = 0; t < T; ++t) col[t] = w4_column(a, column(t) + c16, q, 4 / GS);
    // wave w brings step w of a block: rows past the tile's last repeat it (their results are dropped), and a step past K
    // reads what is there and is masked to zeros, so that every load of the loop is unconditional
    const bool short_k = a.full == 0 && w >= a.rest;
    const uint8_t *xt = (const uint8_t *)a.x + (int64_t)rt.first * a.sh.K * 2;
    uint32_t xo[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = 16 * m + c16 < rt.rows ? 16 * m + c16 : rt.rows - 1;
        xo[m] = (uint32_t)(r * (int)a.sh.K + (short_k ? 0 : 32 * w) + 8 * q) * 2u;
    }
    const int blocks = a.blocks;
    u32x4 xn[2][MT];
    auto bring = [&](int b, int i) {
        const int c = b < blocks ? b : blocks - 1;
        const uint8_t *xb = xt + (int64_t)(c < a.full || w < a.rest ? c : 0) * (2 * kBlockK);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            uint32_t o = xo[m];
            asm volatile("" : "+v"(o));
            xn[i][m] = *(const u32x4 *)(xb + o);
        }
    };
    auto place = [&](int b, int i) {
        const uint32_t mask = b < a.full || w < a.rest ? 0xFFFFFFFFu : 0u;
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[i][w][m][lane] = xn[i][m] & mask;
    };
    f32x4 total[MT][T];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < T; ++t) total[m][t] = f32x4{0, 0, 0, 0};
    W4Block<T, 4 / GS, ZEROS> ring[2];
    auto use = [&](int i) {
        w4_use<DT, MT, T, GS, ZEROS>(ring[i], [&](int m, int s) { return rows[i][s][m][lane]; }, total);
    };
    bring(0, 0);
    ring[0].template fetch<false>(we, col, 0);
    bring(1, 1);
    ring[1].template fetch<false>(we, col, blocks > 1 ? 1 : 0);
    place(0, 0);
    __syncthreads();
    int b = 0;
    for (; b + 1 < blocks; b += 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bring(b + i + 2, i);
            use(i);
            ring[i].template fetch<false>(we, col, b + i + 2 < blocks ? b + i + 2 : blocks - 1);
            place(b + i + 1, 1 - i);
            __syncthreads();
        }
    }
    if (b < blocks) use(0);
    // the sums and the lane's place are taken up anew here: kept in view over the loop, what follows it costs the loop
    // registers (one form spilled ten)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < T; ++t) asm volatile("" : "+v"(total[m][t]));
    int late = lane;
    asm volatile("" : "+v"(late));
    const int row0 = 4 * (late >> 4), col0 = late & 15;
    float poison[4] = {0.0f, 0.0f, 0.0f, 0.0f};              // NaN from the first sum that is not finite on
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) poison[i] = __fmaf_rn(total[m][t][i], 0.0f, poison[i]);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 16 * m + i + row0;
            if (row >= rt.rows) continue;
            uint16_t *o = (uint16_t *)a.out + (int64_t)(rt.first + row) * a.out_cols;
            if (a.swiglu) {
#pragma unroll
                for (int t = 0; t < T; t += 2)
                    if (column(t) + col0 < a.out_cols)
                        o[column(t) + col0] = (uint16_t)to_bits16<DT>(w4_swiglu(total[m][t][i], total[m][t + 1][i]));
            } else {
#pragma unroll
                for (int t = 0; t < T; ++t)
                    if (column(t) + col0 < a.out_cols) o[column(t) + col0] = (uint16_t)to_bits16<DT>(total[m][t][i]);
            }
        }
    }
    if (poison[0] + poison[1] + poison[2] + poison[3] == 0.0f) return;
    uint32_t again = 0;                                      // pairs of tiles, 2p and 2p + 1, with such a sum: m, i, p in the bits
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int p = 0; p < T / 2; ++p)
                if (16 * m + i + row0 < rt.rows && !(w4_finite(total[m][2 * p][i]) && w4_finite(total[m][2 * p + 1][i])))
                    again |= 1u << ((m * 4 + i) * (T / 2) + p);
    for (uint32_t left = again; left; left &= left - 1) {
        const int bit = __builtin_ctz(left), row = bit / (T / 2) / 4 * 16 + bit / (T / 2) % 4 + row0, p = bit % (T / 2);
        const int c0 = column(2 * p) + col0, c1 = column(2 * p + 1) + col0;
        const uint8_t *x = xt + (int64_t)row * a.sh.K * 2;
        uint16_t *o = (uint16_t *)a.out + (int64_t)(rt.first + row) * a.out_cols;
        float v0 = 0.0f;
#pragma unroll 1
        for (int j = 0; j < 2; ++j) {
            const float v = w4_plain<DT, GS, ZEROS>(a, we, j ? c1 : c0, x);
            const int c = j ? c1 : c0;
            if (!a.swiglu && c < a.out_cols) o[c] = (uint16_t)to_bits16<DT>(v);
            if (a.swiglu && j && c0 < a.out_cols) o[c0] = (uint16_t)to_bits16<DT>(w4_swiglu(v0, v));
            v0 = v;
        }
    }
}

// HIP launches up to 2^32 - 1 threads.  The tiled kernel takes 256 for 256 columns of 32 or 64 rows, the few-row kernel 64
// for 32 columns of 16 rows where there are many, so only a great number of experts of a few rows each passes the limit.
static bool w4_fits(int64_t blocks, int threads) { return blocks * threads < (int64_t)1 << 32; }

template <int DT, bool ZEROS>
static int launch_w4(W4Args a, int64_t busy, hipStream_t s) {
    const int64_t P = a.P;
    // row tiles: the most there can be, and one for rows without an expert
    auto tiles = [&](int64_t R) { return busy + (P - busy) / R + 1; };
    const int64_t mean = (P + busy - 1) / busy;
    const int mt = !ZEROS && mean >= 128 ? 4 : 2;
    const int64_t per_wide = kManyTiles * (a.swiglu ? 32 : 64), wide = (a.out_cols + per_wide - 1) / per_wide;
    if (mean > 8 && wide * (tiles(16 * mt) - 1) >= 256) {
        a.col_blocks = (int)wide;
        if (!w4_fits(wide * tiles(16 * mt), 4 * kWave)) return TERRACE_EINVAL;
        const unsigned grid = (unsigned)(wide * tiles(16 * mt));
#define TERRACE_MANY(MT)                                                                            \
    if (a.sh.group == 128) w4_many_kernel<DT, MT, 4, ZEROS><<<grid, 4 * kWave, 0, s>>>(a);          \
    else if (a.sh.group == 64) w4_many_kernel<DT, MT, 2, ZEROS><<<grid, 4 * kWave, 0, s>>>(a);      \
    else w4_many_kernel<DT, MT, 1, ZEROS><<<grid, 4 * kWave, 0, s>>>(a)
        if constexpr (!ZEROS) {
            if (mt == 4) {
                TERRACE_MANY(4);
                return check_launch();
            }
        }
        TERRACE_MANY(2);
#undef TERRACE_MANY
        return check_launch();
    }
    const int64_t sets = a.swiglu ? (a.out_cols + 15) / 16 : (a.out_cols + 31) / 32, n = sets * (tiles(16) - 1);
    a.split = 1;
    while (a.split < kMaxSplit && n * a.split < 4096 && a.full >= 2 * a.split) a.split *= 2;
    const int waves = a.split > 4 ? a.split : 4;
    a.per = (a.full + a.split - 1) / a.split;
    a.sets = waves / a.split;
    a.col_blocks = (int)((sets + a.sets - 1) / a.sets);
    if (!w4_fits(a.col_blocks * tiles(16), waves * kWave)) return TERRACE_EINVAL;
    const unsigned grid = (unsigned)(a.col_blocks * tiles(16)), threads = (unsigned)(waves * kWave);
    if (a.sh.group == 128) w4_few_kernel<DT, 4, ZEROS><<<grid, threads, 0, s>>>(a);
    else if (a.sh.group == 64) w4_few_kernel<DT, 2, ZEROS><<<grid, threads, 0, s>>>(a);
    else w4_few_kernel<DT, 1, ZEROS><<<grid, threads, 0, s>>>(a);
    return check_launch();
}

int run_w4_linear(const void *x, int dtype, int64_t P, const int64_t *counts, const void *codes, const void *scales,
                  const void *zeros, int n_experts, int64_t N, int64_t K, int group, int swiglu, void *out,
                  hipStream_t s) {
    const W4Shape sh{n_experts, N, K, group};
    if (P < 0 || P > ((int64_t)1 << 30) || (dtype != TERRACE_BF16 && dtype != TERRACE_F16) || !sh.ok() || (swiglu && N % 2))
        return TERRACE_EINVAL;
    if (P == 0) return TERRACE_OK;
    if (!x || (!counts && n_experts != 1) || !codes || !scales || !out || (((uintptr_t)x | (uintptr_t)codes) & 15) ||
        (((uintptr_t)scales | (uintptr_t)zeros) & 7) || ((uintptr_t)out & 1))
        return TERRACE_EINVAL;
    const int64_t busy = P < n_experts ? P : n_experts;      // experts that can hold a row
    const int64_t out_cols = swiglu ? N / 2 : N;
    const W4Args a{x, counts, (int)P, sh, (const u32x4 *)codes, (const uint16_t *)scales, (const uint8_t *)zeros, swiglu,
                   out, (int)out_cols, (int)sh.tiles(), (int)sh.blocks(), (int)(K / kBlockK), (int)(K % kBlockK / 32), 1, 1,
                   1, 1};
    if (dtype == TERRACE_BF16)
        return zeros ? launch_w4<TERRACE_BF16, true>(a, busy, s) : launch_w4<TERRACE_BF16, false>(a, busy, s);
    return zeros ? launch_w4<TERRACE_F16, true>(a, busy, s) : launch_w4<TERRACE_F16, false>(a, busy, s);
}

}  // namespace terrace
