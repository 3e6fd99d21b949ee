// va_int4.cu -- 4-bit codes with a scale (and a zero point) per group of columns: the quantizer, and
// the products of up to 16 queries with a table of coded rows.
//
// Stored format (the codes are those of va_sq_quantize_int4, per row): row r holds ceil(dim / 32) * 16
// bytes, element 2i in the low and 2i + 1 in the high nibble of byte i, two's complement [-8, 7],
// padded with zeros; scales and zero points are [n x ceil(dim / group)]. A code c stands for
// scale * (c - zero).
//
// Scores: out[q, r] = xs_q * sum_g scale[r, g] * sum_{j in g} (c[r, j] - zero[r, g]) x[q, j].
// The codes are read once per pass of queries, 4 bits for 2 to 64 operations: HBM-bound, if unpacking keeps
// pace: the logic pipe takes half an instruction per clock and scheduler. The products run on the tensor cores
// through mma.sync (codes are A, 16 rows; queries are B, 8 columns). tcgen05 would need the unpacked codes written
// to shared memory to use a 128-row tile whose columns stay mostly empty. Two forms:
//   * DIGITS, integer m16n8k32: three logic instructions turn 8 codes into 8 bytes c + 8. An int8 query is one
//     column; an fp32 or bf16 query becomes, per group, fixed-point numbers of 62 bits below the power of two above
//     the group's largest |x|, in eight columns of signed 8-bit digits: an element keeps all its bits down to 2^-38 of
//     that |x| (bf16: 2^-54), and below it is off by at most 2^-62 of it. (With 31 bits in four columns, the rest of a
//     group whose outlier meets codes that stand for zero would lose what the outlier leaves no room for.) Group
//     sums are exact integers below 2^22; they start at 1.5 * 2^23 as a bit pattern, less (8 + zero) times the digits'
//     sum, so that the finished accumulator read as fp32 and less 1.5 * 2^23 is the group's sum.
//   * PIECES, bf16 m16n8k16: 11 instructions turn 8 codes into 8 exact bf16 values c - zero. A bf16 query is one
//     column, exact; an fp32 query is split by truncation into three bf16 values of 8 mantissa bits each, exact, that
//     are multiplied in turn into the same sum.
//   Digits cost a column tile and its recombination per group and query, pieces cost more per code: digits serve int8
//   queries and up to two others, pieces the rest (300000 x 1536, group 128, bf16 queries: two as digits 54 us, as pieces
//   68 us; 100000 x 4096, group 32, four fp32 queries with zero points: digits in four tiles 202 us, pieces 175 us).
//   * Logic and issue slots are what remains above the memory time: 2000000 x 768 with one query takes 134 us at the full
//     clock (6.1 TB/s), 155 us once the power cap has lowered it; 16 int8 queries x 300000 x 1536 69 us (41 us of memory).
//   * Group scales and query scales are applied and the groups summed in fp32.
//   * A warp owns 32 rows. Its tiles of 32 rows x 128 bytes arrive by TMA in a ring of its own (one
//     lane issues, the warp waits; no other warp is involved), 128B-swizzled, so that the four words
//     of a 32-code block of 8 rows are one conflict-free access.
//   * The queries are laid out once per block in shared memory in the order the mma reads.
//   * Few rows: WK warps share a row tile, each takes every WK-th 256-code chunk, and the first adds
//     the partial sums in order.
#include <algorithm>

#include "va_tcgen05.cuh"

namespace {

using namespace va::tc;

constexpr int TR = 32;             // rows per warp tile
constexpr int CHUNK = 256;         // codes per ring slot and row (128 bytes)
constexpr int SLOT = TR * 128;     // bytes of a ring slot

struct MatvecArgs {
    const void* x;
    const void* scales;
    const int8_t* zeros;
    const float* x_scales;
    float* out;
    int64_t n, out_stride;
    int row_tiles;
    int dim, groups, nq, x_dtype;  // columns and groups of this launch
    int x_pitch, scale_pitch;      // of a whole query and of a row's scales
    int add;                       // the launch adds to out (a further range of columns)
    int chunks;  // 256-code chunks per row
    int wk;      // warps sharing a row tile
    int ring;    // slots per warp
    int stall;   // -1, or (tests) the copies after which a warp's issuer stops
};

// What a column of B holds: an int8 query; a digit of a query; a query (bf16) or its three pieces in turn (fp32).
enum Mode { DIGITS_INT8, DIGITS_WIDE, BF16, BF16X3 };
constexpr int pieces_of(int mode) { return mode == BF16X3 ? 3 : 1; }
constexpr bool is_bf16(int mode) { return mode == BF16 || mode == BF16X3; }
// Bytes of shared memory that one chunk's queries take per column tile.
constexpr int frag_bytes(int mode) { return 32 * 8 * (is_bf16(mode) ? 16 * pieces_of(mode) : 8); }

constexpr uint32_t MAGIC = 0x4B400000u;  // 1.5 * 2^23 as fp32 bits
constexpr float MAGIC_F = 12582912.f;

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

// The low nibbles of four bytes as c + 8.
__device__ __forceinline__ uint32_t nibbles(uint32_t w) { return (w & 0x0F0F0F0Fu) ^ 0x08080808u; }

// d = a b + c
__device__ __forceinline__ void mma_u8s8(uint32_t (&d)[4], const uint32_t (&a)[4], uint2 b, const uint32_t (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// (w & 0x000F000F) ^ 0x43084308: the nibbles at bits 0 and 16 as bf16 values 128 + (c + 8); less 136 + zero.
__device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t bias) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"((w & 0x000F000Fu) ^ 0x43084308u), "r"(bias));
    return d;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint2 b, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Loads that stay where they are written (ahead of the chunk they are for), as the wait and the products do.
__device__ __forceinline__ uint32_t load_ahead(const uint16_t* p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_ahead(const float* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ int load_ahead(const int8_t* p) {
    int v;
    asm volatile("ld.global.nc.s8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// The scales and zero points that a lane holds of one chunk: of its four rows, groups t and t + 4 of the chunk.
template <typename S, bool ZERO, int GROUP>
struct ChunkScales {
    static constexpr int GPC = CHUNK / GROUP;           // groups per chunk
    static constexpr int SPL = GPC > 4 ? GPC / 4 : 1;   // held per lane and row
    uint32_t sc[4][SPL];  // as stored
    int zp[ZERO ? 4 : 1][ZERO ? SPL : 1];
    __device__ __forceinline__ void load(const MatvecArgs& a, const int64_t (&base)[4], int c, int t) {
#pragma unroll
        for (int p = 0; p < SPL; ++p) {
            const int gi = min(c * GPC + (t & (GPC - 1)) + 4 * p, a.groups - 1);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sc[r][p] = load_ahead(static_cast<const S*>(a.scales) + base[r] + gi);
                if constexpr (ZERO) zp[r][p] = load_ahead(a.zeros + base[r] + gi);
            }
        }
    }
};

// First scales of a lane's four rows in a row tile; rows past the end repeat the last one (they are not stored).
__device__ __forceinline__ void row_bases(const MatvecArgs& a, int tile, int g, int64_t (&base)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) base[r] = min((int64_t)tile * TR + g + 8 * r, a.n - 1) * a.scale_pitch;
}

// What a block keeps of the queries in shared memory.
struct QueryShared {
    uint2* frag;    // [chunk][block 8][step 2 of bf16][NT][piece][lane]: in the mma's order
    int* start;     // [group][NT * 8]: MAGIC - 8 * sum of the column's digits
    float* weight;  // [group][NT][4]: of a query's pairs of columns (DIGITS_WIDE)
};

// Eight elements of query q from column j on (zeros where there are none) as fp32. The vector form needs queries that start on 16 (int8: 8) bytes and whole vectors.
__device__ __forceinline__ void load_query(const MatvecArgs& a, int q, int j, bool vector, float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
    if (q >= a.nq || j >= a.dim) return;
    const int64_t at = (int64_t)q * a.x_pitch + j;
    if (a.x_dtype == VA_DTYPE_F32) {
        const float* x = static_cast<const float*>(a.x) + at;
        if (vector) {
            const float4 u = __ldg(reinterpret_cast<const float4*>(x)), v = __ldg(reinterpret_cast<const float4*>(x) + 1);
            f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = v.x, f[5] = v.y, f[6] = v.z, f[7] = v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < a.dim) f[k] = __ldg(x + k);
        }
    } else if (a.x_dtype == VA_DTYPE_BF16) {
        const uint16_t* x = static_cast<const uint16_t*>(a.x) + at;
        if (vector) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(x));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(k & 1 ? w[k >> 1] & 0xFFFF0000u : w[k >> 1] << 16);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < a.dim) f[k] = va::bf2f(__ldg(x + k));
        }
    } else {
        const int8_t* x = static_cast<const int8_t*>(a.x) + at;
        if (vector) {
            const int2 u = __ldg(reinterpret_cast<const int2*>(x));
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = (float)(int8_t)((k < 4 ? u.x : u.y) >> (8 * (k & 3)));
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < a.dim) f[k] = (float)__ldg(x + k);
        }
    }
}

__device__ __forceinline__ uint32_t high_halves(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

// One warp lays out chunk c of query q: lane 4b + t has the 8 elements of word t of 32-code block b.
template <int NT, int GROUP, int MODE>
__device__ __forceinline__ void lay_out(const MatvecArgs& a, const QueryShared& sh, int q, int c, bool vector, int lane) {
    float f[8];
    load_query(a, q, c * CHUNK + lane * 8, vector, f);
    const int blk = c * 8 + (lane >> 2), t = lane & 3;
    if constexpr (is_bf16(MODE)) {
        // k16 step h of a block pairs the nibbles (2h, 2h + 4) and (2h + 1, 2h + 5) of each word.
        constexpr int P = pieces_of(MODE);
        bool finite[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) finite[k] = fabsf(f[k]) < INFINITY;
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                sh.frag[((((size_t)blk * 2 + h) * NT + (q >> 3)) * P + p) * 32 + (q & 7) * 4 + t] =
                    make_uint2(high_halves(f[2 * h], f[2 * h + 4]), high_halves(f[2 * h + 1], f[2 * h + 5]));
            if constexpr (P > 1) {
                // what truncation left for the next piece; an infinity or a NaN stays in the first
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    f[k] = finite[k] ? f[k] - __uint_as_float(__float_as_uint(f[k]) & 0xFFFF0000u) : 0.f;
            }
        }
    } else {
        constexpr int LANES = GROUP / 8;  // of a group
        constexpr bool wide = MODE == DIGITS_WIDE;
        constexpr int planes = wide ? 8 : 1;
        const int grp = (c * CHUNK + lane * 8) / GROUP;
        uint32_t v[8][wide ? 2 : 1];  // (low and high word)
        if constexpr (wide) {
            float top = 0.f;
            int finite = 1;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                finite &= fabsf(f[k]) < INFINITY;
                top = fmaxf(top, fabsf(f[k]));
            }
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) {
                finite &= __shfl_xor_sync(0xFFFFFFFFu, finite, o);
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            }
            // 2^e > top; the fixed point's unit is 2^(e - 62), not below the smallest fp32. (The factor may
            // exceed fp32: two steps.)
            const auto power = [](int n) { return __int_as_float((n + 127) << 23); };
            const int e = max((int)(__float_as_uint(top) >> 23) - 126, -87);
            const float up = power((62 - e) / 2), up2 = power(62 - e - (62 - e) / 2);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                // With 128 added to each byte but the highest, no digit is below zero: the bytes are the digits, plus 128.
                const long long u = (finite ? __float2ll_rn(f[k] * up * up2) : 0) + 0x0080808080808080ll;
                v[k][0] = (uint32_t)u;
                v[k][1] = (uint32_t)(u >> 32);
            }
            if (lane % LANES == 0) {
                const float w = finite ? power(e - 14) : __int_as_float(0x7FC00000);
                *reinterpret_cast<float4*>(sh.weight + ((size_t)grp * NT + q) * 4) =
                    make_float4(w, w * 0x1p-16f, w * 0x1p-16f * 0x1p-16f, w * 0x1p-16f * 0x1p-16f * 0x1p-16f);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k][0] = (uint32_t)(int)f[k];
        }
#pragma unroll
        for (int p = 0; p < planes; ++p) {  // column 0 has the highest digit
            constexpr int LAST = planes - 1;
            const int col = q * planes + p, word = (LAST - p) / 4;
            const uint32_t byte = (LAST - p) & 3, pick = byte | ((byte + 4) << 4);
            uint32_t d[2];  // even and odd elements
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                d[o] = __byte_perm(__byte_perm(v[o][word], v[2 + o][word], pick), __byte_perm(v[4 + o][word], v[6 + o][word], pick), 0x5410);
                if (wide && p > 0) d[o] ^= 0x80808080u;
            }
            sh.frag[((size_t)blk * NT + (col >> 3)) * 32 + (col & 7) * 4 + t] = make_uint2(d[0], d[1]);
            int sum = __dp4a((int)d[0], 0x01010101, __dp4a((int)d[1], 0x01010101, 0));
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (lane % LANES == 0) sh.start[(size_t)grp * NT * 8 + col] = (int)(MAGIC - 8u * (uint32_t)sum);
        }
    }
}

// NT column tiles of 8; S = scale type (uint16_t: bf16); GROUP = 32, 64, 128.
template <int MODE, int NT, int WARPS, typename S, bool ZERO, int GROUP>
__global__ void __launch_bounds__(WARPS * 32, 1)
    k_int4_matvec(const __grid_constant__ CUtensorMap codes, MatvecArgs a, int* err, uint64_t limit_ns) {
    extern __shared__ uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    using Scales = ChunkScales<S, ZERO, GROUP>;
    constexpr int GPC = Scales::GPC, P = pieces_of(MODE);
    constexpr bool WIDE = MODE == DIGITS_WIDE;
    const int groups_pad = a.chunks * GPC;
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = smem + (size_t)warp * a.ring * SLOT;
    QueryShared sh;
    sh.frag = (uint2*)(smem + (size_t)WARPS * a.ring * SLOT);
    sh.start = (int*)(sh.frag + (size_t)a.chunks * NT * (frag_bytes(MODE) / 8));
    sh.weight = (float*)(sh.start + (is_bf16(MODE) ? 0 : (size_t)groups_pad * NT * 8));
    uint64_t* bars = (uint64_t*)(sh.weight + (is_bf16(MODE) ? 0 : (size_t)groups_pad * NT * 4));
    uint64_t* full = bars + warp * a.ring;
    volatile int* s_abort = (volatile int*)(bars + WARPS * a.ring);
    float* join = (float*)(bars + WARPS * a.ring + 1);  // [WARPS][NT * 8][32], only with wk > 1

    const int teams = WARPS / a.wk, team = warp / a.wk, part = warp % a.wk;
    // Row tiles go round the blocks first, so that few tiles spread over all SMs.
    const int first = team * (int)gridDim.x + (int)blockIdx.x, step = (int)gridDim.x * teams;
    const int mine = (a.chunks - part + a.wk - 1) / a.wk;  // chunks of this warp per row tile
    const int tiles = first < a.row_tiles ? (a.row_tiles - first + step - 1) / step : 0;

    if (lane == 0) {
        for (int s = 0; s < a.ring; ++s) mbar_init(&full[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) *s_abort = 0;
    __syncwarp();
    // Position of the next load to issue (lane 0): slot, row tile and chunk.
    int64_t left = a.stall < 0 ? (int64_t)tiles * mine : min((int64_t)tiles * mine, (int64_t)a.stall);
    int issue_tile = first, issue_chunk = part;
    auto issue = [&](int s) {
        mbar_expect_tx(&full[s], SLOT);
        tma_load_2d(ring + (size_t)s * SLOT, &codes, &full[s], issue_chunk * 128, issue_tile * TR);
        --left;
        issue_chunk += a.wk;
        if (issue_chunk >= a.chunks) {
            issue_chunk = part;
            issue_tile += step;
        }
    };
    if (lane == 0)
        for (int i = 0; i < a.ring && left > 0; ++i) issue(i);
    Scales next;
    int64_t base[4];
    row_bases(a, min(first, a.row_tiles - 1), g, base);
    next.load(a, base, part, t);

    constexpr int QUERIES = WIDE ? NT : NT * 8;
    const int item = a.x_dtype == VA_DTYPE_F32 ? 4 : a.x_dtype == VA_DTYPE_BF16 ? 2 : 1;
    const bool vector = a.dim % 8 == 0 && a.x_pitch % 8 == 0 && ((uintptr_t)a.x & (item == 1 ? 7 : 15)) == 0;
    for (int i = warp; i < a.chunks * QUERIES; i += WARPS) lay_out<NT, GROUP, MODE>(a, sh, i % QUERIES, i / QUERIES, vector, lane);
    __syncthreads();

    // (the 16-byte unit b of row r lies at unit b ^ (r & 7) of its 128 bytes)
    const uint32_t slot0 = smem_u32(ring) + g * 128 + g * 16 + t * 4;
    const uint2* const frag0 = sh.frag + lane;
    bool dead = false;
    int s = 0;
    uint32_t phase = 0;
    // After a wait for chunk c of tile k has expired: copies in flight, those issued and not yet used, write this block's
    // shared memory, so it stays until they have landed. None is issued after that.
    const auto settle = [&](int k, int c) {
        const int per_tile = (a.chunks - part + a.wk - 1) / a.wk;
        const int64_t all = (int64_t)tiles * per_tile, copies = a.stall < 0 ? all : min(all, (int64_t)a.stall);
        const int flying = (int)(copies - left - ((int64_t)k * per_tile + (c - part) / a.wk));
        for (int i = s; i < s + flying; ++i)
            mbar_drain(&full[i < a.ring ? i : i - a.ring], i < a.ring ? phase : phase ^ 1u, kDrainLimitNs);
    };
    constexpr int ACC = WIDE ? 2 : 4;  // sums per row tile half: rows g and g + 8, of a pair of columns each or added up
    for (int k = 0; k < tiles; ++k) {
        const int tile = first + k * step;
        float acc[NT][2][ACC];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < ACC; ++i) acc[n][m][i] = 0.f;
        for (int c = part; c < a.chunks; c += a.wk) {
            // The next chunk's scales are on their way while this one is multiplied.
            const Scales now = next;
            if (c + a.wk < a.chunks) {
                next.load(a, base, c + a.wk, t);
            } else if (k + 1 < tiles) {
                row_bases(a, tile + step, g, base);
                next.load(a, base, part, t);
            }
            // Every lane waits: the phase it has seen is what makes the copy's bytes visible to it.
            if (!dead && __any_sync(0xFFFFFFFFu, !mbar_wait(&full[s], phase, s_abort, err, limit_ns))) {
                dead = true;
                if (lane == 0) settle(k, c);
            }
            if (dead) break;
            const uint32_t slot = slot0 + s * SLOT;
            const uint2* fr = frag0 + (size_t)c * NT * (frag_bytes(MODE) / 8);
            const int2* starts = reinterpret_cast<const int2*>(sh.start + (size_t)c * GPC * NT * 8) + t;
            const float* weight = sh.weight + (size_t)c * GPC * NT * 4 + t;
#pragma unroll
            for (int gi = 0; gi < GPC; ++gi) {
                float gs[4];
                int zero[4];
                const int from = (lane & ~3) | (gi & 3);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    gs[r] = __uint_as_float(__shfl_sync(0xFFFFFFFFu, now.sc[r][Scales::SPL > 1 ? gi >> 2 : 0], from)
                                            << (sizeof(S) == 2 ? 16 : 0));
                    zero[r] = 0;
                    if constexpr (ZERO) zero[r] = __shfl_sync(0xFFFFFFFFu, now.zp[r][Scales::SPL > 1 ? gi >> 2 : 0], from);
                }
                if constexpr (is_bf16(MODE)) {
                    float grp[NT][2][4];
                    uint32_t bias[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) bias[r] = (0x4308u + (uint32_t)zero[r]) * 0x10001u;
#pragma unroll
                    for (int b = 0; b < GROUP / 32; ++b) {
                        const int blk = gi * (GROUP / 32) + b;
                        uint32_t w[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) w[r] = lds32((slot ^ (blk << 4)) + r * 1024);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t f[2][4];
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                f[r >> 1][r & 1] = pair(w[r] >> (8 * h), bias[r]);
                                f[r >> 1][2 + (r & 1)] = pair(w[r] >> (8 * h + 4), bias[r]);
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int p = 0; p < P; ++p) {
                                    const uint2 q = fr[(((blk * 2 + h) * NT + n) * P + p) * 32];
                                    const float none[4] = {0.f, 0.f, 0.f, 0.f};
                                    if (b + h + p == 0) {
                                        mma_bf16(grp[n][0], f[0], q, none);
                                        mma_bf16(grp[n][1], f[1], q, none);
                                    } else {
                                        mma_bf16(grp[n][0], f[0], q, grp[n][0]);
                                        mma_bf16(grp[n][1], f[1], q, grp[n][1]);
                                    }
                                }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int i = 0; i < ACC; ++i) acc[n][m][i] = fmaf(gs[2 * m + (i >> 1)], grp[n][m][i], acc[n][m][i]);
                } else {
                    uint32_t grp[NT][2][4];
#pragma unroll
                    for (int b = 0; b < GROUP / 32; ++b) {
                        const int blk = gi * (GROUP / 32) + b;
                        uint32_t f[2][4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t w = lds32((slot ^ (blk << 4)) + r * 1024);
                            f[r >> 1][r & 1] = nibbles(w);
                            f[r >> 1][2 + (r & 1)] = nibbles(w >> 4);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint2 q = fr[(blk * NT + n) * 32];
                            if (b == 0) {
                                const int2 d = starts[(gi * NT + n) * 4];
                                uint32_t start[2][4];
#pragma unroll
                                for (int m = 0; m < 2; ++m)
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        start[m][i] = (uint32_t)(i & 1 ? d.y : d.x) -
                                                      (ZERO ? (uint32_t)(zero[2 * m + (i >> 1)] * ((int)(MAGIC - (uint32_t)(i & 1 ? d.y : d.x)) >> 3)) : 0u);
                                mma_u8s8(grp[n][0], f[0], q, start[0]);
                                mma_u8s8(grp[n][1], f[1], q, start[1]);
                            } else {
                                mma_u8s8(grp[n][0], f[0], q, grp[n][0]);
                                mma_u8s8(grp[n][1], f[1], q, grp[n][1]);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float w = WIDE ? weight[(gi * NT + n) * 4] : 0.f;
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            float v[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(grp[n][m][i]) - MAGIC_F;
#pragma unroll
                            for (int i = 0; i < ACC; ++i) {
                                if constexpr (WIDE)
                                    acc[n][m][i] = fmaf(gs[2 * m + i], fmaf(v[2 * i], 256.f, v[2 * i + 1]) * w, acc[n][m][i]);
                                else
                                    acc[n][m][i] = fmaf(gs[2 * m + (i >> 1)], v[i], acc[n][m][i]);
                            }
                        }
                    }
                }
            }
            __syncwarp();  // the slot is free: every lane has read it
            if (lane == 0 && left > 0) issue(s);
            if (++s == a.ring) {
                s = 0;
                phase ^= 1u;
            }
        }
        if (a.wk > 1) {
            // Partial sums of the team's other warps, added in warp order.
            float* at = join + (size_t)warp * NT * 8 * 32 + lane;
            if (part > 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < ACC; ++i) at[((n * 2 + m) * ACC + i) * 32] = acc[n][m][i];
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(a.wk * 32) : "memory");
            if (part == 0) {
                for (int p = 1; p < a.wk; ++p) {
                    const float* from = at + (size_t)p * NT * 8 * 32;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int i = 0; i < ACC; ++i) acc[n][m][i] += from[((n * 2 + m) * ACC + i) * 32];
                }
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(a.wk * 32) : "memory");
        }
        if (part == 0 && !dead) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const int64_t row = (int64_t)tile * TR + g + 16 * m + 8 * hi;
                        if constexpr (WIDE) {
                            // Lane t holds digits 2t and 2t + 1 of query n.
                            float v = acc[n][m][hi];
                            v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
                            v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
                            if (t == 0 && row < a.n && n < a.nq) a.out[(int64_t)n * a.out_stride + row] = v;
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int q = n * 8 + 2 * t + i;
                                if (row < a.n && q < a.nq) {
                                    float* const to = a.out + (int64_t)q * a.out_stride + row;
                                    float v = acc[n][m][2 * hi + i];
                                    if constexpr (MODE == DIGITS_INT8) {
                                        if (a.x_scales) v *= __ldg(a.x_scales + q);
                                    } else if constexpr (MODE == BF16X3) {
                                        if (a.add) v += *to;
                                    }
                                    *to = v;
                                }
                            }
                        }
                    }
        }
    }
}

// Warps per block: what the registers allow (128 a thread at 16 warps).
constexpr int warps_of(int nt) { return nt == 4 ? 8 : 16; }

struct Launch {
    CUtensorMap codes;
    MatvecArgs a;
    int group, scale_dtype, grid;
    size_t smem;
};

template <int MODE, int NT, typename S, bool ZERO, int GROUP>
int launch_matvec(va_context* ctx, const Launch& l) {
    constexpr auto kern = k_int4_matvec<MODE, NT, warps_of(NT), S, ZERO, GROUP>;
    VA_TRY(va_kernel_once<kern>(ctx->device, kMaxBlockSmem));
    kern<<<l.grid, warps_of(NT) * 32, l.smem, ctx->stream>>>(l.codes, l.a, ctx->d_error, wait_limit_ns(ctx->timeout_ms));
    return va_check_launch("k_int4_matvec");
}

template <int MODE, int NT, typename S, bool ZERO>
int launch_group(va_context* ctx, const Launch& l) {
    if (l.group == 32) return launch_matvec<MODE, NT, S, ZERO, 32>(ctx, l);
    if (l.group == 64) return launch_matvec<MODE, NT, S, ZERO, 64>(ctx, l);
    return launch_matvec<MODE, NT, S, ZERO, 128>(ctx, l);
}

template <int MODE, int NT>
int launch_types(va_context* ctx, const Launch& l) {
    if (l.scale_dtype == VA_DTYPE_BF16)
        return l.a.zeros ? launch_group<MODE, NT, uint16_t, true>(ctx, l) : launch_group<MODE, NT, uint16_t, false>(ctx, l);
    return l.a.zeros ? launch_group<MODE, NT, float, true>(ctx, l) : launch_group<MODE, NT, float, false>(ctx, l);
}

// A pass: its mode, column tiles, queries, and chunks of columns per launch.
struct Pass {
    int mode, nt, nq, chunks;
};

// fp32 and bf16 queries: up to two as digits (a column tile each), more as pieces, 8 queries a column tile; three
// pieces of 8 queries leave the ring two slots up to 1536 dimensions: wider rows are taken in equal ranges of columns,
// each launch adding to the scores of the one before. int8 queries: 8 a column tile, up to four. Two tiles of bf16 pieces
// take twice the memory of one, which is left to the ring above 2048 dimensions.
Pass pass_of(int x_dtype, int left, int chunks) {
    if (x_dtype == VA_DTYPE_INT8) {
        const int nt = left > 16 ? 4 : left > 8 ? 2 : 1;
        return Pass{DIGITS_INT8, nt, std::min(left, nt * 8), chunks};
    }
    if (left <= 2) return Pass{DIGITS_WIDE, left, left, chunks};
    if (x_dtype == VA_DTYPE_BF16) {
        const int nt = left > 8 && chunks <= 8 ? 2 : 1;
        return Pass{BF16, nt, std::min(left, nt * 8), chunks};
    }
    const int ranges = (chunks + 5) / 6;
    return Pass{BF16X3, 1, std::min(left, 8), (chunks + ranges - 1) / ranges};
}

int launch_pass(va_context* ctx, const Pass& p, const Launch& l) {
    switch (p.mode) {
        case DIGITS_INT8:
            return p.nt == 1   ? launch_types<DIGITS_INT8, 1>(ctx, l)
                   : p.nt == 2 ? launch_types<DIGITS_INT8, 2>(ctx, l)
                               : launch_types<DIGITS_INT8, 4>(ctx, l);
        case DIGITS_WIDE:
            return p.nt == 1 ? launch_types<DIGITS_WIDE, 1>(ctx, l) : launch_types<DIGITS_WIDE, 2>(ctx, l);
        case BF16:
            return p.nt == 1 ? launch_types<BF16, 1>(ctx, l) : launch_types<BF16, 2>(ctx, l);
        default:
            return launch_types<BF16X3, 1>(ctx, l);
    }
}

// ------------------------------------------------------------------------------------------------
// Quantizer and its inverse: a thread per 8 neighbouring elements (a 32-bit word of codes), GROUP / 8 lanes a group.
// Bound by instructions, not by memory: 1000000 x 768, groups of 64: 796 us from fp32 (67% of the copy rate), 845 us from bf16
// (35%), back to fp32 866 us (61%). (64 registers for a fourth block per SM: 897 us.)
// ------------------------------------------------------------------------------------------------
struct GroupArgs {
    const void* x;
    int64_t n, x_stride;
    int dim, groups, stride;  // stride: bytes of a code row
    int scale_dtype;
    uint8_t* codes;
    void* scales;
    int8_t* zeros;
};

// Eight elements as loaded, those from `n` on zero. ALIGNED: p is on a 16-byte boundary.
template <typename T, bool ALIGNED>
struct Raw8 {
    uint4 q[sizeof(T) / 2];
    T x[8];
    __device__ __forceinline__ void load(const T* p, int n) {
        if (ALIGNED) {
            if (n >= 8) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
                return;
            }
            T last[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) last[e] = e < n ? p[e] : (T)0;
            memcpy(q, last, sizeof(q));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = e < n ? p[e] : (T)0;
        }
    }
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (!ALIGNED) {
            if constexpr (sizeof(T) == 2)
                return va::bf2f(x[e]);
            else
                return x[e];
        } else {
            constexpr int PER = 16 / sizeof(T);
            const uint4 u = q[e / PER];
            const int k = e % PER * sizeof(T) / 4;
            const uint32_t w = k == 0 ? u.x : k == 1 ? u.y : k == 2 ? u.z : u.w;
            return __uint_as_float(sizeof(T) == 4 ? w : e & 1 ? w & 0xFFFF0000u : w << 16);
        }
    }
};

template <typename T, int GROUP, bool ALIGNED>
__global__ void __launch_bounds__(256) k_sq_q4_groups(GroupArgs a) {
    constexpr int LANES = GROUP / 8;
    const int l = threadIdx.x & (LANES - 1);
    const int64_t total = a.n * a.groups, step = (int64_t)gridDim.x * (256 / LANES), row_step = step / a.groups;
    const int group_step = (int)(step % a.groups);
    int64_t i = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES, row = i / a.groups;
    int grp = (int)(i % a.groups);
    // The elements of the next round are on their way while a round is worked on (1000000 x 768 bf16: 953 us without).
    Raw8<T, ALIGNED> next;
    int next_j0 = grp * GROUP + l * 8, next_n = i < total ? a.dim - next_j0 : 0;
    next.load(static_cast<const T*>(a.x) + row * a.x_stride + next_j0, next_n);
    // The lanes of a warp run the same number of rounds.
    for (int64_t i0 = i - (threadIdx.x & 31) / LANES; i0 < total; i0 += step, i += step) {
        const bool live = i < total;
        const int j0 = next_j0, n = next_n;
        const int64_t at = row * a.stride + j0 / 2;
        const Raw8<T, ALIGNED> v = next;
        row += row_step;
        grp += group_step;
        if (grp >= a.groups) {
            grp -= a.groups;
            ++row;
        }
        next_j0 = grp * GROUP + l * 8;
        next_n = i + step < total ? a.dim - next_j0 : 0;
        next.load(static_cast<const T*>(a.x) + row * a.x_stride + next_j0, next_n);
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo = fminf(lo, v[e]);
            hi = fmaxf(hi, v[e]);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        }
        // (halves: hi - lo itself may leave fp32's range; the same bits otherwise, above the scales' floor)
        float s = a.zeros ? __fdiv_rn(fmaf(hi, 0.5f, -0.5f * lo), 7.5f) : __fdiv_rn(fmaxf(-lo, hi), 7.f);
        s = fmaxf(s, 1e-8f);
        // The codes are those of the scale as it is stored.
        if (a.scale_dtype == VA_DTYPE_BF16) s = va::bf2f(va::f2bf_rn(s));
        const float z = a.zeros ? fminf(7.f, fmaxf(-8.f, rintf(-8.f - __fdiv_rn(lo, s)))) : 0.f;
        if (live && l == 0) {
            if (a.scale_dtype == VA_DTYPE_BF16)
                static_cast<uint16_t*>(a.scales)[i] = va::f2bf_rn(s);
            else
                static_cast<float*>(a.scales)[i] = s;
            if (a.zeros) a.zeros[i] = (int8_t)z;
        }
        // x / s + z through the reciprocal is within 2^-18 of the rounded quotient's; adding 1.5 * 2^23 rounds it. Where it
        // lies within 2^-14 of a border between two codes the quotient decides; on the border, where a scale and rows of
        // bf16 meet often (1000000 x 768: 919 us with eight divisions there), the even code.
        const float inv = __frcp_rn(s);
        constexpr float NEAR = 0.5f - 0x1p-14f;
        float off = 0.f;
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = fminf(7.f, fmaxf(-8.f, fmaf(v[e], inv, z))), r = t + MAGIC_F;
            off = fmaxf(off, fabsf(t - (r - MAGIC_F)));
            word |= (__float_as_uint(r) & 0xFu) << (4 * e);
        }
        if (off > NEAR) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = fminf(7.f, fmaxf(-8.f, fmaf(v[e], inv, z))), r = (t + MAGIC_F) - MAGIC_F, d = t - r;
                if (fabsf(d) > NEAR) {
                    const float border = r + copysignf(0.5f, d);
                    int c;
                    if (fmaf(z - border, s, v[e]) == 0.f)
                        c = 2 * (int)rintf(0.5f * border);
                    else
                        c = (int)fminf(7.f, fmaxf(-8.f, rintf(__fdiv_rn(v[e], s) + z)));
                    word = (word & ~(0xFu << (4 * e))) | (uint32_t)(c & 0xF) << (4 * e);
                }
            }
        }
        if (n < 8) word = n <= 0 ? 0u : word & ((1u << (4 * n)) - 1u);  // padding holds zeros
        if (live && j0 < 2 * a.stride) *reinterpret_cast<uint32_t*>(a.codes + at) = word;
    }
}

// The words of a warp stand for one run of the output, whatever the dimension: it goes through shared memory to whole
// lines (700000 x 1001: 2930 us when each thread stores its own).
__global__ void __launch_bounds__(256) k_sq_dq4_groups(GroupArgs a, int group, float* __restrict__ out) {
    __shared__ float s_run[8][256 + 8];  // element p at p + p / 32: no two lanes of a warp meet in a bank
    float* run = s_run[threadIdx.x >> 5];
    const int lane = threadIdx.x & 31, words = (a.dim + 7) / 8;
    const int64_t total = a.n * words, step = (int64_t)gridDim.x * 256, row_step = step / words;
    const int word_step = (int)(step % words);
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / words;
    int word = (int)(i % words);
    struct Word {
        uint32_t codes;
        float scale;
        int zero;
    } next{};
    const auto load = [&] {
        const int64_t g = row * a.groups + word * 8 / group;
        next.codes = *reinterpret_cast<const uint32_t*>(a.codes + row * a.stride + word * 4);
        next.scale = a.scale_dtype == VA_DTYPE_BF16 ? va::bf2f(static_cast<const uint16_t*>(a.scales)[g])
                                                    : static_cast<const float*>(a.scales)[g];
        next.zero = a.zeros ? a.zeros[g] : 0;
    };
    if (i < total) load();
    for (int64_t i0 = i - lane; i0 < total; i0 += step, i += step) {
        const Word w = next;
        const int n = i < total ? min(8, a.dim - word * 8) : 0;
        const int64_t at = row * a.dim + word * 8;
        row += row_step;
        word += word_step;
        if (word >= words) {
            word -= words;
            ++row;
        }
        if (i + step < total) load();
        const int64_t first = __shfl_sync(0xFFFFFFFFu, at, 0);
        const int end = __shfl_sync(0xFFFFFFFFu, (int)(at - first) + n, (int)min((int64_t)31, total - 1 - i0));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int p = (int)(at - first) + e;
            if (e < n) run[p + (p >> 5)] = (float)(((int)(w.codes << (28 - 4 * e)) >> 28) - w.zero) * w.scale;
        }
        __syncwarp();
        for (int p = lane; p < end; p += 32) out[first + p] = run[p + (p >> 5)];
        __syncwarp();
    }
}

template <typename T, bool ALIGNED>
int launch_q4(va_context* ctx, const GroupArgs& a, int group) {
    const int64_t blocks = (a.n * a.groups * (group / 8) + 255) / 256;
    const int grid = (int)std::min<int64_t>(blocks, (int64_t)ctx->sm_count * 8);
    if (group == 32)
        k_sq_q4_groups<T, 32, ALIGNED><<<grid, 256, 0, ctx->stream>>>(a);
    else if (group == 64)
        k_sq_q4_groups<T, 64, ALIGNED><<<grid, 256, 0, ctx->stream>>>(a);
    else
        k_sq_q4_groups<T, 128, ALIGNED><<<grid, 256, 0, ctx->stream>>>(a);
    return va_check_launch("k_sq_q4_groups");
}

// The checks the three entry points share.
int check_table(int64_t n, int dim, int group, int scale_dtype, const void* codes, const void* scales) {
    VA_REQUIRE(n >= 0 && n <= 0x7FFFFFE0, "rows must be in 0..2147483616, got %lld", (long long)n);
    VA_REQUIRE(dim > 0 && dim <= VA_MAX_DIM, "dimension must be in 1..%d, got %d", VA_MAX_DIM, dim);
    VA_REQUIRE(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128, got %d", group);
    VA_REQUIRE(scale_dtype == VA_DTYPE_F32 || scale_dtype == VA_DTYPE_BF16,
               "scale_dtype must be VA_DTYPE_F32 or VA_DTYPE_BF16, got %d", scale_dtype);
    VA_REQUIRE(((uintptr_t)codes & 15) == 0, "codes must be aligned to 16 bytes");
    VA_REQUIRE((uintptr_t)scales % (scale_dtype == VA_DTYPE_BF16 ? 2 : 4) == 0, "scales must be aligned to their elements");
    return VA_OK;
}

}  // namespace

extern "C" {

int va_sq_quantize_int4_groups(va_context* ctx, const void* x, int dtype, int64_t n, int dim, int64_t x_stride, int group,
                               int scale_dtype, uint8_t* codes, void* scales, int8_t* zeros) {
    VA_REQUIRE(ctx && (!n || (x && codes && scales)), "ctx, x, codes and scales must not be NULL");
    VA_REQUIRE(dtype == VA_DTYPE_F32 || dtype == VA_DTYPE_BF16, "dtype must be VA_DTYPE_F32 or VA_DTYPE_BF16, got %d",
               dtype);
    VA_TRY(check_table(n, dim, group, scale_dtype, codes, scales));
    VA_REQUIRE(x_stride >= dim, "x_stride must be at least the dimension %d, got %lld", dim, (long long)x_stride);
    VA_REQUIRE((uintptr_t)x % (dtype == VA_DTYPE_BF16 ? 2 : 4) == 0, "x must be aligned to its elements");
    if (!n) return VA_OK;
    const int64_t groups = (dim + group - 1) / group, es = dtype == VA_DTYPE_BF16 ? 2 : 4;
    const VaSpan sx{"x", x, dim * es, n, x_stride * es}, sc{"codes", codes, n * VA_INT4_ROW_BYTES(dim)},
        ss{"scales", scales, n * groups * (scale_dtype == VA_DTYPE_BF16 ? 2 : 4)}, sz{"zeros", zeros, n * groups};
    VA_TRY(va_refuse_overlap(sc, {sx, ss, sz}));
    VA_TRY(va_refuse_overlap(ss, {sx, sz}));
    VA_TRY(va_refuse_overlap(sz, {sx}));
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const GroupArgs a{x, n, x_stride, dim, (dim + group - 1) / group, VA_INT4_ROW_BYTES(dim), scale_dtype, codes, scales, zeros};
    const bool aligned = (uintptr_t)x % 16 == 0 && x_stride * (dtype == VA_DTYPE_BF16 ? 2 : 4) % 16 == 0;
    if (dtype == VA_DTYPE_BF16)
        return aligned ? launch_q4<uint16_t, true>(ctx, a, group) : launch_q4<uint16_t, false>(ctx, a, group);
    return aligned ? launch_q4<float, true>(ctx, a, group) : launch_q4<float, false>(ctx, a, group);
}

int va_sq_dequantize_int4_groups(va_context* ctx, const uint8_t* codes, const void* scales, const int8_t* zeros, int64_t n,
                                 int dim, int group, int scale_dtype, float* out) {
    VA_REQUIRE(ctx && (!n || (codes && scales && out)), "ctx, codes, scales and out must not be NULL");
    VA_TRY(check_table(n, dim, group, scale_dtype, codes, scales));
    VA_REQUIRE(((uintptr_t)out & 3) == 0, "out must be aligned to its elements");
    if (!n) return VA_OK;
    const int64_t groups = (dim + group - 1) / group;
    VA_TRY(va_refuse_overlap({"out", out, n * dim * 4}, {{"codes", codes, n * VA_INT4_ROW_BYTES(dim)},
                                                         {"scales", scales, n * groups * (scale_dtype == VA_DTYPE_BF16 ? 2 : 4)},
                                                         {"zeros", zeros, n * groups}}));
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const GroupArgs a{nullptr, n, 0, dim, (dim + group - 1) / group, VA_INT4_ROW_BYTES(dim), scale_dtype,
                      const_cast<uint8_t*>(codes), const_cast<void*>(scales), const_cast<int8_t*>(zeros)};
    const int grid = (int)std::min<int64_t>((n * ((dim + 7) / 8) + 255) / 256, (int64_t)ctx->sm_count * 8);
    k_sq_dq4_groups<<<grid, 256, 0, ctx->stream>>>(a, group, out);
    return va_check_launch("k_sq_dq4_groups");
}

int va_int4_matvec(va_context* ctx, const void* x, int x_dtype, const float* x_scales, int nq, const uint8_t* codes,
                   const void* scales, const int8_t* zeros, int64_t n, int dim, int group, int scale_dtype, float* out,
                   int64_t out_stride) {
    VA_REQUIRE(ctx && (!n || !nq || (x && codes && scales && out)), "ctx, x, codes, scales and out must not be NULL");
    VA_REQUIRE(x_dtype == VA_DTYPE_F32 || x_dtype == VA_DTYPE_BF16 || x_dtype == VA_DTYPE_INT8,
               "query dtype must be VA_DTYPE_F32, VA_DTYPE_BF16 or VA_DTYPE_INT8, got %d", x_dtype);
    VA_REQUIRE(!x_scales || x_dtype == VA_DTYPE_INT8, "query scales go with VA_DTYPE_INT8 queries");
    VA_REQUIRE(nq >= 0, "numQueries must not be negative, got %d", nq);
    VA_TRY(check_table(n, dim, group, scale_dtype, codes, scales));
    VA_REQUIRE(nq <= 1 || out_stride >= n, "out_stride must be at least the %lld rows, got %lld", (long long)n,
               (long long)out_stride);
    const size_t es = x_dtype == VA_DTYPE_F32 ? 4 : x_dtype == VA_DTYPE_BF16 ? 2 : 1;
    VA_REQUIRE((uintptr_t)x % es == 0 && (uintptr_t)out % 4 == 0 && (uintptr_t)x_scales % 4 == 0,
               "queries, query scales and out must be aligned to their elements");
    if (!n || !nq) return VA_OK;
    const int64_t all_groups = n * ((dim + group - 1) / group);
    VA_TRY(va_refuse_overlap({"out", out, n * 4, nq, out_stride * 4},
                             {{"the queries", x, (int64_t)nq * dim * (int64_t)es}, {"the query scales", x_scales, (int64_t)nq * 4},
                              {"codes", codes, n * VA_INT4_ROW_BYTES(dim)},
                              {"scales", scales, all_groups * (scale_dtype == VA_DTYPE_BF16 ? 2 : 4)}, {"zeros", zeros, all_groups}}));
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);

    const auto enc = get_encode_fn();
    if (!enc) return va_set_error(VA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    Launch l{};
    l.group = group;
    l.scale_dtype = scale_dtype;
    MatvecArgs& a = l.a;
    a.n = n;
    a.out_stride = out_stride;
    a.row_tiles = (int)((n + TR - 1) / TR);
    a.x_pitch = dim;
    a.scale_pitch = (dim + group - 1) / group;
    a.x_dtype = x_dtype;
    a.stall = test_stall_tiles();
    const int chunks = (dim + CHUNK - 1) / CHUNK;
    l.grid = std::min(ctx->sm_count, a.row_tiles);
    int mapped = -1;  // the chunk at which the tensor map starts
    const auto codes_from = [&](int chunk) {
        if (chunk == mapped) return VA_OK;
        mapped = chunk;
        const cuuint64_t pitch = VA_INT4_ROW_BYTES(dim);
        const cuuint64_t dims[2] = {pitch - (cuuint64_t)chunk * (CHUNK / 2), (cuuint64_t)n};
        const cuuint32_t box[2] = {CHUNK / 2, TR}, estr[2] = {1, 1};
        const CUresult r = enc(&l.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes) + (size_t)chunk * (CHUNK / 2), dims,
                               &pitch, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return va_set_error(VA_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
        return VA_OK;
    };
    for (int q0 = 0; q0 < nq; q0 += a.nq) {
        const Pass p = pass_of(x_dtype, nq - q0, chunks);
        a.nq = p.nq;
        a.x_scales = x_scales ? x_scales + q0 : nullptr;
        a.out = out + (int64_t)q0 * out_stride;
        for (int c0 = 0; c0 < chunks; c0 += p.chunks) {
            // Chunks c0 .. c0 + a.chunks - 1 of every row.
            const int g0 = c0 * (CHUNK / group);
            VA_TRY(codes_from(c0));
            a.chunks = std::min(p.chunks, chunks - c0);
            a.dim = std::min(dim - c0 * CHUNK, a.chunks * CHUNK);
            a.groups = (a.dim + group - 1) / group;
            a.add = c0 > 0;
            a.x = static_cast<const uint8_t*>(x) + ((size_t)q0 * dim + (size_t)c0 * CHUNK) * es;
            a.scales = static_cast<const uint8_t*>(scales) + (size_t)g0 * (scale_dtype == VA_DTYPE_BF16 ? 2 : 4);
            a.zeros = zeros ? zeros + g0 : nullptr;
            // Warps per row tile: what leaves the busiest warp the least to do, a tile's end counted as half a chunk and a
            // join as one and a half.
            const int warps = warps_of(p.nt);
            double best = 0;
            for (int wk = 1; wk <= 8 && wk <= a.chunks; wk *= 2) {
                const int64_t slots = (int64_t)l.grid * (warps / wk);
                const double cost = (double)((a.row_tiles + slots - 1) / slots) * ((a.chunks + wk - 1) / wk + (wk > 1 ? 2.0 : 0.5));
                if (wk == 1 || cost < best) {
                    best = cost;
                    a.wk = wk;
                }
            }
            const size_t queries = (size_t)p.nt * a.chunks * (frag_bytes(p.mode) + (is_bf16(p.mode) ? 0 : CHUNK / group * (8 + 4) * 4));
            const size_t rest = 1024 + queries + 16 + (a.wk > 1 ? (size_t)warps * p.nt * 8 * 32 * 4 : 0);
            a.ring = (int)std::min<size_t>(6, (227 * 1024 - rest) / (warps * (SLOT + 8)));
            l.smem = rest + (size_t)a.ring * warps * (SLOT + 8);
            VA_TRY(launch_pass(ctx, p, l));
        }
    }
    return VA_OK;
}

}  // extern "C"
