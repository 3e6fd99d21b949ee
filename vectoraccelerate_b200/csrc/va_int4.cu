// va_int4.cu -- 4-bit codes with a scale (and a zero point) per group of columns: the quantizer, and
// the products of up to 16 queries with a table of coded rows.
//
// Stored format (the codes are those of va_sq_quantize_int4, per row): row r holds ceil(dim / 32) * 16
// bytes, element 2i in the low and 2i + 1 in the high nibble of byte i, two's complement [-8, 7],
// padded with zeros; scales and zero points are [n x ceil(dim / group)]. A code c stands for
// scale * (c - zero).
//
// Scores: out[q, r] = xs_q * sum_g scale[r, g] * sum_{j in g} (c[r, j] - zero[r, g]) x[q, j].
// The codes are read once per pass of up to 32 columns, 4 bits for 2 to 32 operations: HBM-bound, if
// unpacking keeps pace. So the products run on the tensor cores through mma.sync m16n8k16 (codes are A, 16
// rows; queries are B, 8 columns): a code costs 1.4 integer instructions to become an exact bf16 and
// nothing more for 1..8 columns, where fp32 FMAs would take 1.5 + columns. tcgen05 would need the
// unpacked codes written to shared memory (4 bytes of traffic per byte read) to use a 128-row tile
// whose columns stay mostly empty.
//   * The codes enter as integers in [-15, 15] (exact in bf16), the scale multiplies the fp32 group sum.
//   * bf16 and int8 queries are exact as one bf16 column; an fp32 query is split by truncation into
//     three bf16 columns of 8 mantissa bits each, exact again, and the three sums are added at the end.
//   * A warp owns 32 rows. Its tiles of 32 rows x 128 bytes arrive by TMA in a ring of its own (one
//     lane issues, the warp waits; no other warp is involved), 128B-swizzled, so that the four words
//     of a 32-code block of 8 rows are one conflict-free access.
//   * The query fragments are laid out once per block in shared memory in the order the mma reads.
//   * Few rows: WK warps share a row tile, each takes every WK-th 256-code chunk, and the first adds
//     the partial sums in order.
#include <algorithm>

#include "va_tcgen05.cuh"

namespace {

using namespace va::tc;

constexpr int TR = 32;             // rows per warp tile
constexpr int CHUNK = 256;         // codes per ring slot and row (128 bytes)
constexpr int SLOT = TR * 128;     // bytes of a ring slot
constexpr int MAX_NT = 4;          // column tiles of 8 per pass

struct MatvecArgs {
    const void* x;
    const void* scales;
    const int8_t* zeros;
    const float* x_scales;
    float* out;
    int64_t n, out_stride;
    int row_tiles;
    int dim, group, groups, nq, x_dtype;
    int chunks;  // 256-code chunks per row
    int wk;      // warps sharing a row tile
    int ring;    // slots per warp
};

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

// (w & 0x000F000F) ^ 0x43084308: the two nibbles at bits 0 and 16 as bf16 values 128 + (c + 8).
__device__ __forceinline__ uint32_t nibbles(uint32_t w) { return (w & 0x000F000Fu) ^ 0x43084308u; }

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Column `col` of the query operand at element j: the query's value, or piece col & 3 of an fp32
// query (three pieces of 8 mantissa bits, the fourth column is zero). bf16 bit pattern.
__device__ __forceinline__ uint16_t query_bits(const MatvecArgs& a, int col, int j) {
    if (j >= a.dim) return 0;
    if (a.x_dtype == VA_DTYPE_F32) {
        const int q = col >> 2, piece = col & 3;
        if (q >= a.nq || piece == 3) return 0;
        float v = static_cast<const float*>(a.x)[(int64_t)q * a.dim + j];
        uint32_t u = __float_as_uint(v) & 0xFFFF0000u;
        if ((u & 0x7F800000u) == 0x7F800000u) {  // infinity or NaN: all of it in the first piece
            if (v != v) u |= 0x00400000u;
            return piece == 0 ? (uint16_t)(u >> 16) : (uint16_t)0;
        }
        for (int p = 0; p < piece; ++p) {
            v -= __uint_as_float(u);
            u = __float_as_uint(v) & 0xFFFF0000u;
        }
        return (uint16_t)(u >> 16);
    }
    if (col >= a.nq) return 0;
    const int64_t at = (int64_t)col * a.dim + j;
    if (a.x_dtype == VA_DTYPE_BF16) return static_cast<const uint16_t*>(a.x)[at];
    return (uint16_t)(__float_as_uint((float)static_cast<const int8_t*>(a.x)[at]) >> 16);
}

template <typename S>
__device__ __forceinline__ float scale_of(const S* p) {
    if constexpr (sizeof(S) == 2)
        return va::bf2f(__ldg(p));
    else
        return __ldg(p);
}

// The scales (and 136 + zero point, as bf16 bits) that a lane holds of one chunk: of its four rows, groups t and
// t + 4 of the chunk.
template <typename S, bool ZERO, int GROUP>
struct ChunkScales {
    static constexpr int GPC = CHUNK / GROUP;           // groups per chunk
    static constexpr int SPL = GPC > 4 ? GPC / 4 : 1;   // held per lane and row
    float sc[4][SPL];
    uint32_t zp[ZERO ? 4 : 1][ZERO ? SPL : 1];
    __device__ __forceinline__ void load(const MatvecArgs& a, int64_t row0, int c, int g, int t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // rows past the end repeat the last one: they are not stored
            const int64_t base = min(row0 + g + 8 * r, a.n - 1) * a.groups;
#pragma unroll
            for (int p = 0; p < SPL; ++p) {
                const int gi = min(c * GPC + (t & (GPC - 1)) + 4 * p, a.groups - 1);
                sc[r][p] = scale_of(static_cast<const S*>(a.scales) + base + gi);
                if constexpr (ZERO) zp[r][p] = 0x4308u + (uint32_t)(int)__ldg(a.zeros + base + gi);
            }
        }
    }
};

// NT column tiles of 8; S = scale type (uint16_t: bf16); GROUP = 32, 64, 128.
template <int NT, int WARPS, typename S, bool ZERO, int GROUP>
__global__ void __launch_bounds__(WARPS * 32, 1)
    k_int4_matvec(const __grid_constant__ CUtensorMap codes, MatvecArgs a, int* err, uint64_t limit_ns) {
    extern __shared__ uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = smem + (size_t)warp * a.ring * SLOT;
    uint2* frag = (uint2*)(smem + (size_t)WARPS * a.ring * SLOT);  // [chunk][step 16][NT][lane]
    uint64_t* bars = (uint64_t*)(frag + (size_t)a.chunks * 16 * NT * 32);
    uint64_t* full = bars + warp * a.ring;
    volatile int* s_abort = (volatile int*)(bars + WARPS * a.ring);
    float* join = (float*)(bars + WARPS * a.ring + 1);  // [WARPS][NT][2][4][32], only with wk > 1

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
    int64_t left = (int64_t)tiles * mine;
    uint32_t issued = 0;  // counted to the ring's length only
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
        for (; issued < (uint32_t)a.ring && left > 0; ++issued) issue((int)issued);
    using Scales = ChunkScales<S, ZERO, GROUP>;
    Scales next;
    if (tiles > 0) next.load(a, (int64_t)first * TR, part, g, t);

    // Query fragments. k16 step i of a chunk: half i & 1 of 32-code block i >> 1. Lane (g, t) reads word
    // t of the block, whose nibbles 0..7 are elements 8t..8t+7; half h pairs the nibbles (2h, 2h + 4) and
    // (2h + 1, 2h + 5), which B's registers must match for column g.
    for (int e = threadIdx.x; e < a.chunks * 16 * NT * 32; e += WARPS * 32) {
        const int l = e & 31, nt = (e >> 5) % NT, i = (e >> 5) / NT;
        const int j = (i >> 1) * 32 + (l & 3) * 8 + 2 * (i & 1), col = nt * 8 + (l >> 2);
        uint2 f;
        f.x = query_bits(a, col, j) | ((uint32_t)query_bits(a, col, j + 4) << 16);
        f.y = query_bits(a, col, j + 1) | ((uint32_t)query_bits(a, col, j + 5) << 16);
        frag[e] = f;
    }
    __syncthreads();

    const uint32_t slot0 = smem_u32(ring) + g * 128 + t * 4;
    bool dead = false;
    int s = 0;
    uint32_t phase = 0;
    for (int k = 0; k < tiles; ++k) {
        const int tile = first + k * step;
        const int64_t row0 = (int64_t)tile * TR;
        float acc[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][m][i] = 0.f;
        for (int c = part; c < a.chunks; c += a.wk) {
            // The next chunk's scales are on their way while this one is multiplied.
            const Scales now = next;
            const bool last = c + a.wk >= a.chunks;
            if (!last || k + 1 < tiles) next.load(a, last ? row0 + (int64_t)step * TR : row0, last ? part : c + a.wk, g, t);
            // Every lane waits: the phase it has seen is what makes the copy's bytes visible to it.
            if (!dead) dead = __any_sync(0xFFFFFFFFu, !mbar_wait(&full[s], phase, s_abort, err, limit_ns));
            if (dead) break;
            const uint32_t slot = slot0 + s * SLOT;
            const uint2* fr = frag + (size_t)c * 16 * NT * 32 + lane;
#pragma unroll
            for (int gi = 0; gi < Scales::GPC; ++gi) {
                float grp[NT][2][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) grp[n][m][i] = 0.f;
                float gs[4];
                uint32_t bias[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int from = (lane & ~3) | (gi & 3);
                    gs[r] = __shfl_sync(0xFFFFFFFFu, now.sc[r][Scales::SPL > 1 ? gi >> 2 : 0], from);
                    if constexpr (ZERO) {
                        const uint32_t z = __shfl_sync(0xFFFFFFFFu, now.zp[r][Scales::SPL > 1 ? gi >> 2 : 0], from);
                        bias[r] = z | (z << 16);  // 136 + zero point, exact in bf16
                    } else {
                        bias[r] = 0x43084308u;  // 136
                    }
                }
#pragma unroll
                for (int b = 0; b < GROUP / 32; ++b) {
                    const int blk = gi * (GROUP / 32) + b;
                    uint32_t w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[r] = lds32(slot + r * 1024 + ((blk ^ g) << 4));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t f[2][4];
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            f[m][0] = sub_bf16x2(nibbles(w[2 * m] >> (8 * h)), bias[2 * m]);
                            f[m][1] = sub_bf16x2(nibbles(w[2 * m + 1] >> (8 * h)), bias[2 * m + 1]);
                            f[m][2] = sub_bf16x2(nibbles(w[2 * m] >> (8 * h + 4)), bias[2 * m]);
                            f[m][3] = sub_bf16x2(nibbles(w[2 * m + 1] >> (8 * h + 4)), bias[2 * m + 1]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint2 q = fr[((blk * 2 + h) * NT + n) * 32];
                            mma_bf16(grp[n][0], f[0], q.x, q.y);
                            mma_bf16(grp[n][1], f[1], q.x, q.y);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(gs[2 * m + (i >> 1)], grp[n][m][i], acc[n][m][i]);
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
                        for (int i = 0; i < 4; ++i) at[((n * 2 + m) * 4 + i) * 32] = acc[n][m][i];
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
                            for (int i = 0; i < 4; ++i) acc[n][m][i] += from[((n * 2 + m) * 4 + i) * 32];
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
                        const int64_t row = row0 + g + 16 * m + 8 * hi;
                        const float v0 = acc[n][m][2 * hi], v1 = acc[n][m][2 * hi + 1];
                        if (a.x_dtype == VA_DTYPE_F32) {
                            // Columns 4q..4q+3 are pieces of query q: lanes t = 0, 1 hold query 2n, t = 2, 3 query 2n + 1.
                            float v = v0 + v1;
                            v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
                            const int q = n * 2 + (t >> 1);
                            if ((t & 1) == 0 && row < a.n && q < a.nq) a.out[(int64_t)q * a.out_stride + row] = v;
                        } else {
                            const int q = n * 8 + 2 * t;
                            if (row < a.n) {
                                if (q < a.nq) a.out[(int64_t)q * a.out_stride + row] = a.x_scales ? v0 * __ldg(a.x_scales + q) : v0;
                                if (q + 1 < a.nq)
                                    a.out[(int64_t)(q + 1) * a.out_stride + row] = a.x_scales ? v1 * __ldg(a.x_scales + q + 1) : v1;
                            }
                        }
                    }
        }
    }
    // After an expired wait: copies still in flight write this block's shared memory. Of slot i the last
    // copy issued completes phase `phase` (slots from s on) or the next one (slots already reissued).
    if (dead && lane == 0)
        for (int i = 0; i < a.ring && i < (int)issued; ++i)
            mbar_drain(&full[i], i >= s ? phase : phase ^ 1u, kDrainLimitNs);
}

// Warps per block: what the registers allow (128 a thread at 16 warps).
constexpr int warps_of(int nt) { return nt == 4 ? 8 : 16; }

template <int NT, typename S, bool ZERO, int GROUP>
int launch_matvec(va_context* ctx, const CUtensorMap& codes, const MatvecArgs& a, int grid, size_t smem) {
    auto kern = k_int4_matvec<NT, warps_of(NT), S, ZERO, GROUP>;
    VA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kern<<<grid, warps_of(NT) * 32, smem, ctx->stream>>>(codes, a, ctx->d_error, wait_limit_ns(ctx->timeout_ms));
    return va_check_launch("k_int4_matvec");
}

template <int NT, typename S, bool ZERO>
int launch_group(va_context* ctx, const CUtensorMap& codes, const MatvecArgs& a, int grid, size_t smem) {
    if (a.group == 32) return launch_matvec<NT, S, ZERO, 32>(ctx, codes, a, grid, smem);
    if (a.group == 64) return launch_matvec<NT, S, ZERO, 64>(ctx, codes, a, grid, smem);
    return launch_matvec<NT, S, ZERO, 128>(ctx, codes, a, grid, smem);
}

template <int NT>
int launch_types(va_context* ctx, const CUtensorMap& codes, const MatvecArgs& a, int scale_dtype, int grid, size_t smem) {
    if (scale_dtype == VA_DTYPE_BF16)
        return a.zeros ? launch_group<NT, uint16_t, true>(ctx, codes, a, grid, smem)
                       : launch_group<NT, uint16_t, false>(ctx, codes, a, grid, smem);
    return a.zeros ? launch_group<NT, float, true>(ctx, codes, a, grid, smem)
                   : launch_group<NT, float, false>(ctx, codes, a, grid, smem);
}

// ------------------------------------------------------------------------------------------------
// Quantizer and its inverse: 16 lanes per (row, group), GROUP / 16 neighbouring elements a lane.
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

template <typename T>
__device__ __forceinline__ float value_of(const T* p) {
    if constexpr (sizeof(T) == 2)
        return va::bf2f(*p);
    else
        return *p;
}

template <typename T, int GROUP>
__global__ void __launch_bounds__(256) k_sq_q4_groups(GroupArgs a) {
    constexpr int E = GROUP / 16;
    const int l = threadIdx.x & 15;
    const int64_t total = a.n * a.groups;
    for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4; i < (total + 1) / 2 * 2;
         i += ((int64_t)gridDim.x * blockDim.x) >> 4) {
        const bool live = i < total;  // the two halves of a warp run the same number of rounds
        const int64_t row = (live ? i : total - 1) / a.groups;
        const int grp = (int)((live ? i : total - 1) % a.groups), j0 = grp * GROUP + l * E;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        float v[E], lo = 0.f, hi = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = j0 + e < a.dim ? value_of(x + j0 + e) : 0.f;
            lo = fminf(lo, v[e]);
            hi = fmaxf(hi, v[e]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        }
        float s = a.zeros ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(-lo, hi), 7.f);
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
        uint8_t* out = a.codes + row * a.stride;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const int b = (j0 + e) >> 1;
            if (!live || b >= a.stride) continue;
            int c[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                c[k] = j0 + e + k < a.dim ? (int)fminf(7.f, fmaxf(-8.f, rintf(__fdiv_rn(v[e + k], s) + z))) : 0;
            out[b] = (uint8_t)((c[0] & 0xF) | ((c[1] & 0xF) << 4));
        }
    }
}

__global__ void __launch_bounds__(256) k_sq_dq4_groups(GroupArgs a, int group, float* __restrict__ out) {
    const int64_t total = a.n * a.dim;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / a.dim;
        const int j = (int)(i % a.dim);
        const int64_t g = row * a.groups + j / group;
        const int nib = (a.codes[row * a.stride + (j >> 1)] >> (4 * (j & 1))) & 0xF;
        const int c = (nib ^ 8) - 8;
        const float s = a.scale_dtype == VA_DTYPE_BF16 ? va::bf2f(static_cast<const uint16_t*>(a.scales)[g])
                                                       : static_cast<const float*>(a.scales)[g];
        out[i] = (float)(c - (a.zeros ? (int)a.zeros[g] : 0)) * s;
    }
}

template <typename T>
int launch_q4(va_context* ctx, const GroupArgs& a, int group) {
    const int64_t blocks = (a.n * a.groups + 15) / 16;
    const int grid = (int)std::min<int64_t>(blocks, (int64_t)ctx->sm_count * 8);
    if (group == 32)
        k_sq_q4_groups<T, 32><<<grid, 256, 0, ctx->stream>>>(a);
    else if (group == 64)
        k_sq_q4_groups<T, 64><<<grid, 256, 0, ctx->stream>>>(a);
    else
        k_sq_q4_groups<T, 128><<<grid, 256, 0, ctx->stream>>>(a);
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
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const GroupArgs a{x, n, x_stride, dim, (dim + group - 1) / group, VA_INT4_ROW_BYTES(dim), scale_dtype, codes, scales, zeros};
    return dtype == VA_DTYPE_BF16 ? launch_q4<uint16_t>(ctx, a, group) : launch_q4<float>(ctx, a, group);
}

int va_sq_dequantize_int4_groups(va_context* ctx, const uint8_t* codes, const void* scales, const int8_t* zeros, int64_t n,
                                 int dim, int group, int scale_dtype, float* out) {
    VA_REQUIRE(ctx && (!n || (codes && scales && out)), "ctx, codes, scales and out must not be NULL");
    VA_TRY(check_table(n, dim, group, scale_dtype, codes, scales));
    if (!n) return VA_OK;
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const GroupArgs a{nullptr, n, 0, dim, (dim + group - 1) / group, VA_INT4_ROW_BYTES(dim), scale_dtype,
                      const_cast<uint8_t*>(codes), const_cast<void*>(scales), const_cast<int8_t*>(zeros)};
    const int grid = (int)std::min<int64_t>((n * dim + 255) / 256, (int64_t)ctx->sm_count * 8);
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
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);

    const auto enc = get_encode_fn();
    if (!enc) return va_set_error(VA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)VA_INT4_ROW_BYTES(dim), (cuuint64_t)n};
    const cuuint64_t strides[1] = {(cuuint64_t)VA_INT4_ROW_BYTES(dim)};
    const cuuint32_t box[2] = {128, TR}, estr[2] = {1, 1};
    const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return va_set_error(VA_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);

    MatvecArgs a{};
    a.scales = scales;
    a.zeros = zeros;
    a.n = n;
    a.out_stride = out_stride;
    a.row_tiles = (int)((n + TR - 1) / TR);
    a.dim = dim;
    a.group = group;
    a.groups = (dim + group - 1) / group;
    a.x_dtype = x_dtype;
    a.chunks = (dim + CHUNK - 1) / CHUNK;
    const int cols_per_query = x_dtype == VA_DTYPE_F32 ? 4 : 1;
    for (int q0 = 0; q0 < nq;) {
        // Column tiles of this pass: what the queries fill, within 64 KB of fragments (128 KB at 8 warps).
        int nt = 1;
        while (nt < MAX_NT && nt * 8 < (nq - q0) * cols_per_query && 2 * nt * a.chunks <= (nt == 2 ? 32 : 16)) nt *= 2;
        a.nq = std::min(nq - q0, nt * 8 / cols_per_query);
        a.x = static_cast<const uint8_t*>(x) + (size_t)q0 * dim * es;
        a.x_scales = x_scales ? x_scales + q0 : nullptr;
        a.out = out + (int64_t)q0 * out_stride;
        const int warps = warps_of(nt);
        // Warps per row tile: more only while the row tiles leave warps of the grid idle.
        a.wk = 1;
        while (a.wk < 8 && a.wk * 2 <= a.chunks && (int64_t)a.row_tiles * a.wk * 2 <= (int64_t)ctx->sm_count * warps) a.wk *= 2;
        const size_t frag = (size_t)a.chunks * 16 * nt * 32 * sizeof(uint2);
        const size_t rest = 1024 + frag + 16 + (a.wk > 1 ? (size_t)warps * nt * 8 * 32 * 4 : 0);
        a.ring = (int)std::min<size_t>(6, (227 * 1024 - rest) / (warps * (SLOT + 8)));
        const size_t smem = rest + (size_t)a.ring * warps * (SLOT + 8);
        const int grid = std::min(ctx->sm_count, a.row_tiles);
        if (nt == 1)
            VA_TRY(launch_types<1>(ctx, map, a, scale_dtype, grid, smem));
        else if (nt == 2)
            VA_TRY(launch_types<2>(ctx, map, a, scale_dtype, grid, smem));
        else
            VA_TRY(launch_types<4>(ctx, map, a, scale_dtype, grid, smem));
        q0 += a.nq;
    }
    return VA_OK;
}

}  // extern "C"
