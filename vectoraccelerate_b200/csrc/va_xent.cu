// va_xent.cu -- softmax cross entropy of tokens against all rows of a table, and its gradients, on the
// tensor cores; the logits are never kept.
//
// tokens h [T x D], table w [V x D] (bf16), c = logit_scale:
//   z_tv = c h_t . w_v        lse_t = ln sum_v exp z_tv        loss_t = lse_t - z_{t, label_t}
//   G_tv = c g_t (exp(z_tv - lse_t) - [v = label_t])           dh = G w        dw = G^T h
// with g_t the gradient of loss_t. A token whose label is outside [0, V) has no loss: loss 0, G row 0.
//
// Forward, 2TVD operations: k_xent_scores<FORWARD> walks tiles of tokens x 256 rows (TMA ring, one thread issuing
// tcgen05.mma, two TMEM accumulators) and its epilogue keeps each token's running maximum and sum of
// exponentials (in powers of two) in registers, and sets the label's logit aside; the partial pairs of the row splits are
// joined by k_xent_join.
// Backward, 6TVD: the table is taken in chunks of rows so that G of a chunk (bf16) is at most 512 MB (with 256 MB
// the last, partly filled round of tiles weighs more: 2% slower at 8192 x 131072 x 1536).
// k_xent_scores<GRADIENT> recomputes the chunk's logits and stores G; k_xent_grads multiplies it both
// ways, with operands that are contiguous along the wrong axis read as MN-major tiles instead of being
// transposed in memory: dw tiles (M = rows, K = tokens) are finished in one go; dh tiles (M = tokens, K = the
// chunk's rows) add into an fp32 buffer per K split, which k_xent_finish sums and rounds. Where few rows meet many
// tokens dw is split the same way (8192 x 1000 x 64: backward 60 us in one go, 30 split).
// Both directions are compute-bound once T and V pass a few hundred: the tensor pipe and its operand feed are the
// limit. Below D = 256 neither it nor the exponentials (16 per clock and SM) are: 5982 x 6479 x 120 takes 31 us forward, 9 us of
// exponentials and a tensor pipe in use for 18%; the epilogue's instructions and the hand-over of an accumulator every
// two K blocks take the time.
//
// Tiles: a CTA's 128 x 256 tile takes 48 KB of operands per 64 of K, more than shared memory and L2 feed at the
// full rate; a pair of CTAs (cta_group::2) works on 256 x 256 and loads 32 KB each. Measured per chunk of 8192 x
// 16384 x 1536: the two products 797 us with single CTAs, 650 us with pairs. Problems that do not fill the GPU with
// 128-row tiles twice over keep single CTAs, which spread wider; and where even those leave SMs idle, the logits' tiles
// are 128 wide (333 x 5003 x 512: 7.8 us instead of 12.4).
//
// Measured (B200, 8192 x 131072 x 1536): forward 2.4 ms, 1380 TFLOP/s; forward and backward 10.6 ms under the power cap,
// 8TVD at 1240 TFLOP/s, where cuBLAS runs the same three products at 1330; 45 us of it are the four small kernels.
//
// Roundings: G is kept as P - [label] in bf16, without c g_t: a label's entry is then -1 to within its p, where
// c g_t itself would round alike for every token of a mean and bias the gradients by up to 2^-8 (measured: 0.33%
// instead of 0.17% off at 8192 x 131072 x 1536). dh's rows take c g_t when they are finished, in fp32. dw needs it
// inside the sum: h's rows enter as bf16(h c g_t / rho) and dw is multiplied by rho, the largest |c g| of the batch, so that
// equal weights leave h as it is. Everything else is fp32. All orders of summation are fixed.
#include <algorithm>
#include <cmath>

#include "va_tcgen05.cuh"

namespace {

using namespace va::tc;

constexpr int BM = 128;                   // tile rows of a CTA (TMEM lanes)
constexpr int BN = 256;                   // columns of an accumulator
constexpr int BK = 64;                    // elements of K per stage (128 bytes)
constexpr int BOX = 64 * 128;             // bytes of a 64-row box of 128-byte rows
constexpr int A_BYTES = 2 * BOX;
constexpr int RING_BYTES = 4 * 6 * BOX;   // 4 stages of 6 boxes, or 6 stages of 4 (pairs)
constexpr int EPI_BYTES = 32 * 128;       // one staged 32-row x 128-byte piece of an epilogue warp
constexpr int EPI_WARPS = 8;              // two per quarter of the TMEM lanes: each takes half of a tile's columns
constexpr int THREADS = 64 + 32 * EPI_WARPS;  // TMA warp, MMA warp, epilogue warps
constexpr int TMEM_COLS = 512;
constexpr size_t SMEM = 1024 + RING_BYTES + EPI_WARPS * EPI_BYTES + (2 * 6 + 5) * 8 + 16;
// A gradient tile costs its K blocks, but at least this many: its results leave in that time (64 x 100000 x 768: both
// products 84 us with 1, 72 with 2 to 4, 86 with 8).
constexpr int TILE_END = 3;
// Up to this many tokens every block of k_xent_tokens looks for the largest weight among all of them (2 us at most,
// as long as the launch that it saves); beyond, WEIGHT_PARTS blocks do it first.
constexpr int FEW_TOKENS = 2048, WEIGHT_PARTS = 128;
constexpr int64_t G_ENTRIES = 1 << 28;    // gradient entries of a chunk (512 MB of bf16)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

template <bool PAIR>
struct Tile {
    static constexpr int CTAS = PAIR ? 2 : 1;
    static constexpr int M = CTAS * BM;
    static constexpr int STAGES = PAIR ? 6 : 4;
    static constexpr int B_BYTES = (PAIR ? 2 : 4) * BOX;  // a CTA's share of B at the full width
};

enum { FORWARD = 0, GRADIENT = 1 };

// Per token of the backward pass: lse in powers of two, c * g (0: no loss) and the label.
struct TokenGrad {
    float lse2, scale;
    int label, pad;
};

// What the roles of a CTA share. In a pair, CTA 0 leads: its full barriers count both CTAs' bytes, it issues the
// MMAs, and its tempty barriers collect both CTAs' epilogue warps; empty and tfull are signalled in both CTAs.
template <bool PAIR>
struct Roles {
    uint8_t *sA, *sB, *sE;
    uint64_t *full, *empty, *tfull, *tempty, *dbar;
    volatile int* abort_flag;
    uint32_t tmem;
    uint32_t rank;      // in the pair
    int worker, workers;

    __device__ __forceinline__ bool leader() const { return !PAIR || rank == 0; }
    // A bounded wait; one that expires stops the other CTA of the pair too.
    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, uint64_t limit_ns) const {
        if (mbar_wait(bar, parity, abort_flag, err, limit_ns)) return true;
        if constexpr (PAIR) abort_peer(abort_flag, rank);
        return false;
    }
    // Arms stage s for `bytes` of each CTA.
    __device__ __forceinline__ void arm(int s, uint32_t bytes) const {
        if (leader()) mbar_expect_tx(&full[s], bytes * Tile<PAIR>::CTAS);
    }
    __device__ __forceinline__ void load(int s, void* dst, const CUtensorMap* map, int c0, int c1) const {
        if constexpr (PAIR)
            tma_load_2d_pair(dst, map, map_rank(smem_u32(&full[s]), 0), c0, c1);
        else
            tma_load_2d(dst, map, &full[s], c0, c1);
    }
    // Signals a barrier of every CTA once the MMAs issued so far are done.
    __device__ __forceinline__ void commit(uint64_t* bar) const {
        if constexpr (PAIR) {
            mma_commit_pair(map_rank(smem_u32(bar), 0));
            mma_commit_pair(map_rank(smem_u32(bar), 1));
        } else {
            mma_commit(bar);
        }
    }
    // After an abort, before the CTAs rejoin: copies in flight have landed, MMAs issued are done.
    __device__ __forceinline__ void settle_loads(uint32_t issued) const {
        if (!*abort_flag) return;
        if (leader()) drain_loads(full, Tile<PAIR>::STAGES, issued);
        if constexpr (PAIR) settle_ns(1000000ull);
    }
    __device__ __forceinline__ void settle_mmas(bool stalled) const {
        if (!*abort_flag && !stalled) return;
        if constexpr (PAIR)
            mma_commit_pair(map_rank(smem_u32(dbar), 0));
        else
            mma_commit(dbar);
        mbar_drain(dbar, 0u, kDrainLimitNs);
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    // (.ftz: terms below 2^-126 of the largest count as zero)
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// Instruction descriptor: fp32 accumulator, bf16 operands, M rows, N columns; an operand is K-major (0)
// or MN-major (1).
__host__ __device__ constexpr uint32_t idesc_of(int m, int n, int a_mn, int b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// MN-major operand, 128B swizzle: boxes of 64 (MN) x 64 (K), 128 bytes per K row. Groups of 8 K rows are
// 1024 B apart (SBO), neighbouring 64-element blocks of MN one box (LBO). A step of 16 along K is 2048 B.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(BOX >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                 "r"(smem_u32(src)), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                 "r"(smem_u32(src)), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Shared set-up of the two kernels: barriers, TMEM.
template <bool PAIR>
__device__ __forceinline__ Roles<PAIR> set_up(uint8_t* smem_raw) {
    constexpr int STAGES = Tile<PAIR>::STAGES;
    Roles<PAIR> r;
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    r.sA = smem;
    r.sB = smem + (size_t)STAGES * A_BYTES;
    r.sE = smem + RING_BYTES;
    r.full = (uint64_t*)(r.sE + EPI_WARPS * EPI_BYTES);
    r.empty = r.full + STAGES;
    r.tfull = r.empty + STAGES;
    r.tempty = r.tfull + 2;
    r.dbar = r.tempty + 2;
    uint32_t* s_tmem = (uint32_t*)(r.dbar + 1);
    r.abort_flag = (volatile int*)(s_tmem + 1);
    r.rank = PAIR ? cluster_rank() : 0u;
    r.worker = PAIR ? (int)cluster_index() : (int)blockIdx.x;
    r.workers = PAIR ? (int)cluster_count() : (int)gridDim.x;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&r.full[s], 1);
            mbar_init(&r.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&r.tfull[b], 1);
            mbar_init(&r.tempty[b], EPI_WARPS * Tile<PAIR>::CTAS);
        }
        mbar_init(r.dbar, 1);
        *r.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Both CTAs' barriers exist before either CTA signals the other's.
    if constexpr (PAIR) cluster_sync();
    if (threadIdx.x >> 5 == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                         "r"(TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                         "r"(TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    r.tmem = *s_tmem;
    return r;
}

// Every role of every CTA rejoins; TMEM is freed after the last read and the last MMA.
template <bool PAIR>
__device__ __forceinline__ void tear_down(const Roles<PAIR>& r) {
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();
    if (threadIdx.x >> 5 == 1) {
        tc_fence_after();
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(r.tmem), "r"(TMEM_COLS));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(r.tmem), "r"(TMEM_COLS));
    }
}

// Programmatic launches: the next tile kernel of the stream may start its set-up while this kernel runs; before it
// touches global memory it waits for this one to be complete. (So nothing here is read through the read-only path, which
// assumes data that no kernel in flight writes.)
__device__ __forceinline__ void pdl_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A ring position shared by the producer and the MMA issuer.
template <bool PAIR>
struct Ring {
    uint32_t it = 0;
    __device__ __forceinline__ int slot() const { return (int)(it % Tile<PAIR>::STAGES); }
    __device__ __forceinline__ uint32_t phase() const { return (it / Tile<PAIR>::STAGES) & 1u; }
};

// Waits for accumulator `tile`; the whole warp follows lane 0's verdict.
template <bool PAIR>
__device__ __forceinline__ bool wait_accumulator(const Roles<PAIR>& r, uint32_t tile, int lane, int* err, uint64_t limit_ns) {
    int ok = 1;
    if (lane == 0) ok = r.wait(&r.tfull[tile & 1u], (tile >> 1) & 1u, err, limit_ns) ? 1 : 0;
    ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
    tc_fence_after();
    return ok != 0;
}
template <bool PAIR>
__device__ __forceinline__ void release_accumulator(const Roles<PAIR>& r, uint32_t tile, int lane) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) {
        if constexpr (PAIR)
            mbar_arrive_remote(map_rank(smem_u32(&r.tempty[tile & 1u]), 0));
        else
            mbar_arrive(&r.tempty[tile & 1u]);
    }
}

// One lane's 128 bytes of a staged piece: row `lane` of 32, 16-byte units in the 128B swizzle order.
__device__ __forceinline__ void stage_unit(uint8_t* piece, int lane, int unit, uint4 v) {
    *reinterpret_cast<uint4*>(piece + lane * 128 + ((unit ^ (lane & 7)) << 4)) = v;
}

// ------------------------------------------------------------------------------------------------
// Logits: forward statistics, or the gradient of a chunk
// ------------------------------------------------------------------------------------------------
struct ScoreWork {
    int64_t tokens, rows;  // rows: of this launch (the whole table, or one chunk), from row0
    int64_t row0;
    int token_tiles, row_tiles, splits, k_blocks;
    int n;                 // table rows of a tile: 256, or 128 (single CTAs)
    int stall_tiles;       // -1, or (tests) the tiles after which a worker's MMA issuer stops
    float scale2;          // c * log2(e)
    float2* part;          // forward: (maximum of h . w, sum) per [split][column half][token_tiles * tile rows]
    const int64_t* labels; // forward
    float* label_dot;      // forward: h . w of the token's label
    const TokenGrad* tok;  // gradient
};

__device__ __forceinline__ void score_item(const ScoreWork& w, int item, int& tt, int& split, int& r0, int& r1) {
    split = item / w.token_tiles;
    tt = item - split * w.token_tiles;
    r0 = (int)((int64_t)w.row_tiles * split / w.splits);
    r1 = (int)((int64_t)w.row_tiles * (split + 1) / w.splits);
}

// r[i], for an index that is not known to the compiler: halved six times.
__device__ __forceinline__ float pick(const uint32_t (&r)[64], int i) {
    uint32_t v[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) v[k] = i & 32 ? r[k + 32] : r[k];
#pragma unroll
    for (int w = 16; w > 0; w >>= 1)
#pragma unroll
        for (int k = 0; k < w; ++k) v[k] = i & w ? v[k + w] : v[k];
    return __uint_as_float(v[0]);
}

// Running maximum and sum of 2^z over 64 columns of a row, z = acc * scale2; columns at or past
// `valid` do not exist. The maximum is kept as nb = -max z (finite even while no logit was finite), rounded: `sum` is
// relative to 2^-nb as it is.
__device__ __forceinline__ void lse_chunk(uint32_t (&r)[64], float scale2, int valid, float& top, float& nb, float& sum) {
    if (valid < 64) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
            if (i >= valid) r[i] = 0xFF800000u;
    }
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 64; ++i) m[i & 3] = fmaxf(m[i & 3], __uint_as_float(r[i]));
    const float mx = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    if (mx > top) {
        const float was = nb;
        top = mx;
        nb = __fmul_rn(-mx, scale2);
        if (sum != 0.f) sum *= ex2(nb - was);
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 64; ++i) s[i & 3] += ex2(fmaf(__uint_as_float(r[i]), scale2, nb));
    sum += (s[0] + s[1]) + (s[2] + s[3]);
}

// Entries p - [label] of 64 columns of a token, staged as 128 bytes of bf16 (zeros for a token without loss,
// whatever its logits are). `label` is the label's column in the chunk (outside [0, 64): not here); its entry is
// formed in fp32 and replaces the staged one.
__device__ __forceinline__ void grad_chunk(const uint32_t (&r)[64], float scale2, const TokenGrad& tg, int label, uint8_t* piece,
                                           int lane) {
    const uint32_t keep = tg.scale == 0.f ? 0u : 0xFFFFFFFFu;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        uint32_t p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float lo = ex2(fmaf(__uint_as_float(r[u * 8 + k * 2]), scale2, -tg.lse2));
            const float hi = ex2(fmaf(__uint_as_float(r[u * 8 + k * 2 + 1]), scale2, -tg.lse2));
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p[k]) : "f"(hi), "f"(lo));
            p[k] &= keep;
        }
        stage_unit(piece, lane, u, make_uint4(p[0], p[1], p[2], p[3]));
    }
    if ((unsigned)label < 64u) {
        const float z = pick(r, label);
        *reinterpret_cast<uint16_t*>(piece + lane * 128 + ((((unsigned)label >> 3) ^ (lane & 7)) << 4) + (label & 7) * 2) =
            va::f2bf_rn(ex2(fmaf(z, scale2, -tg.lse2)) - 1.f);
    }
}

template <int MODE, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
    k_xent_scores(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                  const __grid_constant__ CUtensorMap map_g, ScoreWork w, int* err, uint64_t limit_ns) {
    extern __shared__ uint8_t smem_raw[];
    pdl_start();
    const Roles<PAIR> r = set_up<PAIR>(smem_raw);
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_items = w.token_tiles * w.splits;
    constexpr int TM = Tile<PAIR>::M;
    const int share = w.n / Tile<PAIR>::CTAS;  // table rows of a tile that this CTA loads
    int tt, split, r0, r1;

    if (warp == 0) {
        if (lane == 0) {
            Ring<PAIR> ring;
            for (int item = r.worker; item < n_items && !*r.abort_flag; item += r.workers) {
                score_item(w, item, tt, split, r0, r1);
                for (int t = r0; t < r1; ++t)
                    for (int kb = 0; kb < w.k_blocks; ++kb, ++ring.it) {
                        const int s = ring.slot();
                        if (!r.wait(&r.empty[s], ring.phase() ^ 1u, err, limit_ns)) goto loads_done;
                        r.arm(s, A_BYTES + share * 128);
                        r.load(s, r.sA + (size_t)s * A_BYTES, &map_h, kb * BK, tt * TM + (int)r.rank * BM);
                        r.load(s, r.sB + (size_t)s * Tile<PAIR>::B_BYTES, &map_w, kb * BK,
                               (int)(w.row0 + (int64_t)t * w.n) + (int)r.rank * share);
                    }
            }
        loads_done:
            r.settle_loads(ring.it);
        }
    } else if (warp == 1) {
        if (lane == 0 && r.leader()) {
            Ring<PAIR> ring;
            uint32_t tile = 0;
            const uint32_t idesc = idesc_of(TM, w.n, 0, 0);
            for (int item = r.worker; item < n_items && !*r.abort_flag; item += r.workers) {
                score_item(w, item, tt, split, r0, r1);
                for (int t = r0; t < r1; ++t, ++tile) {
                    if ((int)tile == w.stall_tiles) goto mma_done;
                    if (!r.wait(&r.tempty[tile & 1u], ((tile >> 1) & 1u) ^ 1u, err, limit_ns)) goto mma_done;
                    tc_fence_after();
                    const uint32_t d = r.tmem + (tile & 1u) * BN;
                    for (int kb = 0; kb < w.k_blocks; ++kb, ++ring.it) {
                        const int s = ring.slot();
                        if (!r.wait(&r.full[s], ring.phase(), err, limit_ns)) goto mma_done;
                        tc_fence_after();
                        const uint32_t a0 = smem_u32(r.sA + (size_t)s * A_BYTES), b0 = smem_u32(r.sB + (size_t)s * Tile<PAIR>::B_BYTES);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma_f16<PAIR>(d, smem_desc(a0 + 32 * j), smem_desc(b0 + 32 * j), idesc, (kb | j) ? 1u : 0u);
                        r.commit(&r.empty[s]);
                    }
                    r.commit(&r.tfull[tile & 1u]);
                }
            }
        mma_done:
            r.settle_mmas(w.stall_tiles >= 0);
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint8_t* piece = r.sE + (size_t)(warp - 2) * EPI_BYTES;
        uint32_t tile = 0;
        for (int item = r.worker; item < n_items; item += r.workers) {
            score_item(w, item, tt, split, r0, r1);
            const int64_t token0 = (int64_t)tt * TM + r.rank * BM + quarter * 32, token = token0 + lane;
            float top = -INFINITY, nb = 0.f, sum = 0.f;
            TokenGrad tg{0.f, 0.f, -1, 0};
            if (token < w.tokens) {
                if constexpr (MODE == GRADIENT) {
                    tg = w.tok[token];
                } else {
                    const int64_t l = w.labels[token];
                    if (l >= 0 && l < w.rows) tg.label = (int)l;
                }
            }
            for (int t = r0; t < r1; ++t, ++tile) {
                if (!wait_accumulator(r, tile, lane, err, limit_ns)) goto epilogue_done;
                const int first = half * (w.n / 2);  // this warp's columns of the tile
                const uint32_t at = r.tmem + ((uint32_t)(quarter * 32) << 16) + (tile & 1u) * BN + first;
                const int64_t col0 = (int64_t)t * w.n + first;
                const int valid = (int)max(min((int64_t)w.n / 2, w.rows - col0), (int64_t)0);
                const int64_t label = (int64_t)tg.label - w.row0 - col0;  // the label's column of this tile half
                // 64 columns at a time, the next ones on their way from TMEM meanwhile.
                const auto use = [&](int c, uint32_t(&v)[64]) {
                    const int at_label = (int)max(min(label, (int64_t)BN) - 64 * c, (int64_t)-1);
                    if constexpr (MODE == FORWARD) {
                        lse_chunk(v, w.scale2, valid - 64 * c, top, nb, sum);
                        if ((unsigned)at_label < 64u) w.label_dot[token] = pick(v, at_label);
                    } else {
                        // the store that last used the piece has read it
                        if (lane == 0) bulk_wait_read<0>();
                        __syncwarp();
                        grad_chunk(v, w.scale2, tg, at_label, piece, lane);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            if (token0 < w.tokens && 64 * c < valid) tma_store_2d(&map_g, piece, (int)(col0 + 64 * c), (int)token0);
                            bulk_commit();
                        }
                    }
                };
                uint32_t ra[64];
                tmem_ld64(at, ra);
                tmem_wait64(ra);
                if (w.n > 128) {
                    uint32_t rb[64];
                    tmem_ld64(at + 64, rb);
                    use(0, ra);
                    tmem_wait64(rb);
                    release_accumulator(r, tile, lane);
                    use(1, rb);
                } else {
                    release_accumulator(r, tile, lane);
                    use(0, ra);
                }
            }
            if constexpr (MODE == FORWARD)
                w.part[((int64_t)split * 2 + half) * w.token_tiles * TM + token] = make_float2(top, sum);
        }
    epilogue_done:
        if (MODE == GRADIENT && lane == 0) bulk_wait_all();
    }
    tear_down(r);
}

// ------------------------------------------------------------------------------------------------
// The two products of a chunk's G
// ------------------------------------------------------------------------------------------------
// Items: n_h = token_tiles * d_tiles * splits of dh (K = a split of the chunk's rows) and n_w = row_tiles *
// d_tiles * splits_w of dw (K = the tokens, or a split of them). A worker is a CTA or a pair.
struct GradWork {
    int64_t row0;           // first table row of the chunk
    int64_t rows;           // rows of the whole table
    int dim;
    int64_t tokens;
    int64_t tokens_pad;     // token_tiles * tile rows: of one split's dh buffer
    int64_t rows_pad;       // row_tiles * tile rows: of one split's dw buffer
    int token_tiles, row_tiles, d_tiles, splits;
    int splits_w;           // K splits of dw; 1: dw is finished at once
    const float* rho;       // what dw is multiplied by
    int n;                  // columns of a tile: 64, 128, 192 or 256 (pairs: 128 or 256)
    int kb_rows, kb_tokens; // K blocks of 64: chunk rows, tokens
    int first;              // first chunk: dh is stored, else added
    int long_h;             // dh items are the longer ones and go out first
    int stall_tiles;        // as in ScoreWork
    int extra;              // shorter items given first to the workers that got one longer item less
};

// The k-th item of worker b, or -1. The longer items go round the workers first; then `extra` shorter
// ones to each worker left with one longer item less (as many as make up for it), then the rest to all.
__device__ __forceinline__ int grad_item(const GradWork& w, int b, int grid, int k, bool& is_h) {
    const int n_h = w.token_tiles * w.d_tiles * w.splits, n_w = w.row_tiles * w.d_tiles * w.splits_w;
    const int n_long = w.long_h ? n_h : n_w, n_short = w.long_h ? n_w : n_h;
    const int over = n_long % grid;
    const int longs = n_long / grid + (b < over ? 1 : 0);
    if (k < longs) {
        is_h = w.long_h;
        return b + k * grid;
    }
    is_h = !w.long_h;
    k -= longs;
    const int late = over ? grid - over : 0;  // workers with one longer item less
    const int given = min(late * w.extra, n_short);
    if (b >= over && late) {
        const int j = (b - over) + k * late;
        if (k < w.extra) {
            if (j < given) return j;
            return -1;  // the shorter items are used up
        }
        k -= w.extra;
    }
    const int64_t j = given + (int64_t)k * grid + (grid - 1 - b);
    return j < n_short ? (int)j : -1;
}

struct GradTile {
    int m, d, kb0, kb1, split;
};
__device__ __forceinline__ GradTile grad_tile(const GradWork& w, int item, bool is_h) {
    GradTile t;
    t.d = item % w.d_tiles;
    const int rest = item / w.d_tiles;
    if (is_h) {
        t.m = rest % w.token_tiles;
        t.split = rest / w.token_tiles;
        t.kb0 = (int)((int64_t)w.kb_rows * t.split / w.splits);
        t.kb1 = (int)((int64_t)w.kb_rows * (t.split + 1) / w.splits);
    } else {
        t.m = rest % w.row_tiles;
        t.split = rest / w.row_tiles;
        t.kb0 = (int)((int64_t)w.kb_tokens * t.split / w.splits_w);
        t.kb1 = (int)((int64_t)w.kb_tokens * (t.split + 1) / w.splits_w);
    }
    return t;
}

template <bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
    k_xent_grads(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_dh,
                 const __grid_constant__ CUtensorMap map_dw, const __grid_constant__ CUtensorMap map_dwp, GradWork w, int* err,
                 uint64_t limit_ns) {
    extern __shared__ uint8_t smem_raw[];
    pdl_start();
    const Roles<PAIR> r = set_up<PAIR>(smem_raw);
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int TM = Tile<PAIR>::M;
    const int boxes = w.n / 64 / Tile<PAIR>::CTAS;  // of B that this CTA loads
    bool is_h;

    if (warp == 0) {
        if (lane == 0) {
            Ring<PAIR> ring;
            for (int k = 0, item; (item = grad_item(w, r.worker, r.workers, k, is_h)) >= 0 && !*r.abort_flag; ++k) {
                const GradTile t = grad_tile(w, item, is_h);
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++ring.it) {
                    const int s = ring.slot();
                    if (!r.wait(&r.empty[s], ring.phase() ^ 1u, err, limit_ns)) goto loads_done;
                    r.arm(s, (2 + boxes) * BOX);
                    uint8_t* a = r.sA + (size_t)s * A_BYTES;
                    uint8_t* b = r.sB + (size_t)s * Tile<PAIR>::B_BYTES;
                    const int m0 = t.m * TM + (int)r.rank * BM, d0 = t.d * w.n + (int)r.rank * boxes * 64;
                    if (is_h) {
                        // A: 128 tokens x 64 chunk rows of G. B: 64 table rows x this CTA's columns.
                        for (int i = 0; i < 2; ++i) r.load(s, a + i * BOX, &map_g, kb * BK, m0 + i * 64);
                        for (int i = 0; i < boxes; ++i) r.load(s, b + i * BOX, &map_w, d0 + i * 64, (int)(w.row0 + kb * BK));
                    } else {
                        // A: 64 tokens x 128 chunk rows of G. B: 64 tokens x this CTA's columns.
                        for (int i = 0; i < 2; ++i) r.load(s, a + i * BOX, &map_g, m0 + i * 64, kb * BK);
                        for (int i = 0; i < boxes; ++i) r.load(s, b + i * BOX, &map_h, d0 + i * 64, kb * BK);
                    }
                }
            }
        loads_done:
            r.settle_loads(ring.it);
        }
    } else if (warp == 1) {
        if (lane == 0 && r.leader()) {
            Ring<PAIR> ring;
            uint32_t tile = 0;
            for (int k = 0, item; (item = grad_item(w, r.worker, r.workers, k, is_h)) >= 0 && !*r.abort_flag; ++k) {
                const GradTile t = grad_tile(w, item, is_h);
                if (t.kb0 >= t.kb1) continue;
                if ((int)tile == w.stall_tiles) goto mma_done;
                if (!r.wait(&r.tempty[tile & 1u], ((tile >> 1) & 1u) ^ 1u, err, limit_ns)) goto mma_done;
                tc_fence_after();
                const uint32_t d = r.tmem + (tile & 1u) * BN;
                const uint32_t idesc = idesc_of(TM, w.n, is_h ? 0 : 1, 1);
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++ring.it) {
                    const int s = ring.slot();
                    if (!r.wait(&r.full[s], ring.phase(), err, limit_ns)) goto mma_done;
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(r.sA + (size_t)s * A_BYTES), b0 = smem_u32(r.sB + (size_t)s * Tile<PAIR>::B_BYTES);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_f16<PAIR>(d, is_h ? smem_desc(a0 + 32 * j) : smem_desc_mn(a0 + 2048 * j), smem_desc_mn(b0 + 2048 * j), idesc,
                                (kb > t.kb0 || j) ? 1u : 0u);
                    r.commit(&r.empty[s]);
                }
                r.commit(&r.tfull[tile & 1u]);
                ++tile;
            }
        mma_done:
            r.settle_mmas(w.stall_tiles >= 0);
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint8_t* piece = r.sE + (size_t)(warp - 2) * EPI_BYTES;
        uint32_t tile = 0;
        const float rho = *w.rho;
        // This warp's columns of a tile, in steps of 64.
        const int c0 = half * ((w.n / 64 + 1) / 2), c1 = half ? w.n / 64 : (w.n / 64 + 1) / 2;
        for (int k = 0, item; (item = grad_item(w, r.worker, r.workers, k, is_h)) >= 0; ++k) {
            const GradTile t = grad_tile(w, item, is_h);
            if (t.kb0 >= t.kb1) continue;
            if (!wait_accumulator(r, tile, lane, err, limit_ns)) break;
            const uint32_t at = r.tmem + ((uint32_t)(quarter * 32) << 16) + (tile & 1u) * BN;
            const int row = t.m * TM + (int)r.rank * BM + quarter * 32;
            // (32 rows behind the last token or row are nobody's)
            const bool none = is_h ? row >= w.tokens : w.row0 + row >= w.rows;
            if (c0 == c1 || none) release_accumulator(r, tile, lane);
            for (int c = none ? c1 : c0; c < c1; ++c) {
                uint32_t v[64];
                tmem_ld64(at + 64 * c, v);
                tmem_wait64(v);
                if (c == c1 - 1) release_accumulator(r, tile, lane);
                const int col = t.d * w.n + 64 * c;
                // fp32: 32 columns a piece; bf16: 64.
                const bool f32 = is_h || w.splits_w > 1;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!f32 && i == 1) break;
                    if (lane == 0) bulk_wait_read<0>();
                    __syncwarp();
                    if (f32) {
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            stage_unit(piece, lane, u, make_uint4(v[32 * i + 4 * u], v[32 * i + 4 * u + 1], v[32 * i + 4 * u + 2], v[32 * i + 4 * u + 3]));
                    } else {
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            uint32_t b[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
                                    : "=r"(b[e])
                                    : "f"(__uint_as_float(v[u * 8 + 2 * e + 1]) * rho), "f"(__uint_as_float(v[u * 8 + 2 * e]) * rho));
                            stage_unit(piece, lane, u, make_uint4(b[0], b[1], b[2], b[3]));
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (f32) {
                            const int at_row = (int)(t.split * (is_h ? w.tokens_pad : w.rows_pad) + row);
                            if (col + 32 * i < w.dim) {
                                if (!is_h)
                                    tma_store_2d(&map_dwp, piece, col + 32 * i, at_row);
                                else if (w.first)
                                    tma_store_2d(&map_dh, piece, col + 32 * i, at_row);
                                else
                                    tma_add_2d(&map_dh, piece, col + 32 * i, at_row);
                            }
                        } else if (col < w.dim) {
                            tma_store_2d(&map_dw, piece, col, (int)(w.row0 + row));
                        }
                        bulk_commit();
                    }
                }
            }
            ++tile;
        }
        if (lane == 0) bulk_wait_all();
    }
    tear_down(r);
}

// ------------------------------------------------------------------------------------------------
// The small kernels around them
// ------------------------------------------------------------------------------------------------
// One warp per token: joins the (maximum, sum) pairs of the splits' halves and forms lse and the loss.
// With m the largest h . w, M = fl(m c log2 e) what its part's sum is relative to and d = m c log2 e - M what M was
// rounded by, lse = c m + ln 2 (log2(sum) - d): the large term is rounded once. The loss takes c (m - h . w_label) in
// its place, with the label's product from the same tile that entered the sum, so that a label which holds nearly all
// of the probability costs no cancellation; what rounding leaves below zero is zero.
__global__ void __launch_bounds__(128)
    k_xent_join(const float2* part, int splits, int64_t pitch, const float* label_dot, const int64_t* labels, int64_t tokens,
                int64_t rows, float scale, float scale2, float* loss, float* lse) {
    pdl_start();
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (t >= tokens) return;
    float top = -INFINITY, sum = 0.f;
    const auto join = [&](float m, float s) {  // (the products are rounded by themselves, as in the parts)
        const float both = fmaxf(top, m), base = __fmul_rn(both, scale2);
        sum = (sum != 0.f ? sum * ex2(__fmul_rn(top, scale2) - base) : 0.f) + (s != 0.f ? s * ex2(__fmul_rn(m, scale2) - base) : 0.f);
        top = both;
    };
    // Eight pairs in flight per lane. (Loads of what the kernel before wrote go to L2.)
    for (int i0 = lane; i0 < splits; i0 += 256) {
        float2 p[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = i0 + 32 * k < splits ? __ldcg(part + (i0 + 32 * k) * pitch + t) : make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (p[k].y != 0.f) join(p[k].x, p[k].y);  // (0: no finite logit there)
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float m = __shfl_xor_sync(0xFFFFFFFFu, top, o), s = __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        join(m, s);
    }
    if (lane == 0) {
        const int64_t label = labels[t];
        const float rest = LN2 * (log2f(sum) - fmaf(top, scale2, -__fmul_rn(top, scale2)));
        lse[t] = sum != 0.f ? fmaf(scale, top, rest) : -INFINITY;
        float l = 0.f;
        if (label >= 0 && label < rows) {
            l = sum != 0.f ? fmaf(scale, top - __ldcg(label_dot + t), rest) : __int_as_float(0x7FC00000);
            l = l < 0.f ? 0.f : l;
        }
        loss[t] = l;
    }
}

__device__ __forceinline__ float token_scale(const int64_t* labels, const float* grad, int64_t t, int64_t rows, float scale) {
    const int64_t label = labels[t];
    return label >= 0 && label < rows ? scale * (grad ? grad[t] : 1.f) : 0.f;
}

// The largest of the numbers (not negative) of a block's threads; all of them get it.
template <int WARPS>
__device__ __forceinline__ float largest_of_block(float m) {
    __shared__ float s_max[WARPS];
    m = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m)));  // (ordered like their bits)
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_max[w]);
    return m;
}

// Many tokens: the largest |c g| of each block's share.
__global__ void __launch_bounds__(256)
    k_xent_weights(const int64_t* labels, const float* grad, int64_t tokens, int64_t rows, float scale, float* part) {
    float m = 0.f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < tokens; i += (int64_t)gridDim.x * 256)
        m = fmaxf(m, fabsf(token_scale(labels, grad, i, rows, scale)));
    m = largest_of_block<8>(m);
    if (threadIdx.x == 0) part[blockIdx.x] = m;
}

// One warp per token: what the backward pass needs of it, and its row of h times c g / rho, with tokens without
// loss set to zero (their rows may hold anything; 0 * NaN would reach the table's gradient). rho is the largest |c g|
// of the batch, so that no quotient is above 1 (where it is not finite, or no token has a loss: 1). It comes from `parts`
// shares, or, with few tokens, from all of them in every block: a launch takes longer than that.
__global__ void __launch_bounds__(128)
    k_xent_tokens(const uint16_t* h, int64_t h_stride, const int64_t* labels, const float* lse, const float* grad, int64_t tokens,
                  int64_t rows, int dim, float scale, const float* part, int parts, TokenGrad* tok, float* rho_out, uint16_t* weighted) {
    pdl_start();
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    float rho = 0.f;
    if (parts) {
        if (threadIdx.x < parts) rho = part[threadIdx.x];
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < (int)tokens; i += 128) rho = fmaxf(rho, fabsf(token_scale(labels, grad, i, rows, scale)));
    }
    rho = largest_of_block<4>(rho);
    if (!(rho > 0.f && rho < INFINITY)) rho = 1.f;
    if (t >= tokens) return;
    const float g = token_scale(labels, grad, t, rows, scale), f = g / rho;
    if (lane == 0) {
        tok[t] = TokenGrad{lse[t] * LOG2E, g, g != 0.f ? (int)labels[t] : -1, 0};
        if (t == 0) *rho_out = rho;
    }
    for (int j = lane * 8; j < dim; j += 256) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (g != 0.f) {
            v = *reinterpret_cast<const uint4*>(h + t * h_stride + j);
            if (f != 1.f) {
                uint32_t* p = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
                        : "=r"(p[k])
                        : "f"(__uint_as_float(p[k] & 0xFFFF0000u) * f), "f"(__uint_as_float(p[k] << 16) * f));
            }
        }
        *reinterpret_cast<uint4*>(weighted + t * dim + j) = v;
    }
}

// Sums K splits in a fixed order, applies the token's c g (dh) or rho (dw, tok NULL) and rounds. `lanes` threads of a
// block take every lanes-th split of the same four elements (few tokens have many splits: 64 x 100000 x 768 18 us with one).
__global__ void __launch_bounds__(256) k_xent_finish(const float4* part, int splits, int lanes, int64_t pitch, int64_t n,
                                                     int per_row, const TokenGrad* tok, const float* rho, uint2* out) {
    __shared__ float4 s_sum[256];
    pdl_start();
    const int per = 256 / lanes, first = threadIdx.x / per;
    for (int64_t b = (int64_t)blockIdx.x * per; b < n; b += (int64_t)gridDim.x * per) {
        const int64_t i = b + threadIdx.x % per;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n) {
            v = part[i + first * pitch];
#pragma unroll 4
            for (int s = first + lanes; s < splits; s += lanes) {
                const float4 u = part[i + s * pitch];
                v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            }
        }
        if (lanes > 1) {
            __syncthreads();
            s_sum[threadIdx.x] = v;
            __syncthreads();
            if (first) continue;
            for (int k = 1; k < lanes; ++k) {
                const float4 u = s_sum[threadIdx.x + k * per];
                v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            }
        }
        if (i >= n) continue;
        const float g = tok ? tok[i / per_row].scale : *rho;
        // (a token without loss has no gradient, whatever the table holds)
        if (tok && g == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
        out[i] = make_uint2(va::f2bf_rn(v.x * g) | ((uint32_t)va::f2bf_rn(v.y * g) << 16),
                            va::f2bf_rn(v.z * g) | ((uint32_t)va::f2bf_rn(v.w * g) << 16));
    }
}

// ------------------------------------------------------------------------------------------------
// Host
// ------------------------------------------------------------------------------------------------
int make_map(CUtensorMap* map, const void* base, bool f32, int64_t cols, int64_t rows, int64_t pitch, int box_cols, int box_rows) {
    const auto enc = get_encode_fn();
    if (!enc) return va_set_error(VA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(pitch * (f32 ? 4 : 2))};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = enc(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                           const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return va_set_error(VA_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return VA_OK;
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A pair's 256-row tiles are worth it when single CTAs would have two tiles each.
bool use_pairs(int sms, int64_t tokens, int64_t rows) {
    return tokens > BM && (tokens + BM - 1) / BM * ((rows + BN - 1) / BN) >= 2 * sms;
}

struct ForwardPlan {
    bool pair;
    int n, token_tiles, row_tiles, splits;
    size_t off_dot, bytes;
};

ForwardPlan plan_forward(int sms, int64_t tokens, int64_t rows) {
    ForwardPlan p;
    p.pair = use_pairs(sms, tokens, rows);
    const int tm = p.pair ? 2 * BM : BM, workers = p.pair ? sms / 2 : sms;
    p.token_tiles = (int)((tokens + tm - 1) / tm);
    // Half as wide tiles where whole ones leave CTAs without work.
    p.n = !p.pair && p.token_tiles * ((rows + BN - 1) / BN) < sms ? BN / 2 : BN;
    p.row_tiles = (int)((rows + p.n - 1) / p.n);
    // Row splits: rounds of the grid x (tiles of an item + half a tile for its start and end).
    double best = 0;
    p.splits = 1;
    for (int sp = 1; sp <= std::min(workers, p.row_tiles); ++sp) {
        const double cost = (double)(((int64_t)p.token_tiles * sp + workers - 1) / workers) * ((p.row_tiles + sp - 1) / sp + 0.5);
        if (sp == 1 || cost <= best) {  // (of equals, the one that uses more workers)
            best = cost;
            p.splits = sp;
        }
    }
    p.off_dot = (size_t)p.splits * 2 * p.token_tiles * tm * sizeof(float2);
    p.bytes = p.off_dot + (size_t)tokens * sizeof(float);
    return p;
}

struct BackwardPlan {
    bool pair;
    int64_t chunk;  // table rows per chunk (a multiple of 256)
    int n_scores;   // tile width of the logits
    int token_tiles, d_tiles, n, splits, splits_w;
    int64_t rows_pad;
    size_t off_rho, off_h, off_dh, off_dw, off_g, bytes;
};

BackwardPlan plan_backward(int sms, int64_t tokens, int64_t rows, int dim) {
    BackwardPlan p;
    p.pair = use_pairs(sms, tokens, rows);
    const int tm = p.pair ? 2 * BM : BM, workers = p.pair ? sms / 2 : sms;
    p.token_tiles = (int)((tokens + tm - 1) / tm);
    p.n_scores = !p.pair && p.token_tiles * ((rows + BN - 1) / BN) < sms ? BN / 2 : BN;
    const int64_t most = std::max<int64_t>(BN, G_ENTRIES / tokens / BN * BN);
    const int64_t chunks = (rows + most - 1) / most;
    p.chunk = up((rows + chunks - 1) / chunks, BN);
    p.d_tiles = (dim + BN - 1) / BN;
    p.n = (int)up((dim + p.d_tiles - 1) / p.d_tiles, p.pair ? 128 : 64);
    // K splits of dh: items of at most half a worker's share of the chunk's work (or 8 K blocks), while
    // the fp32 buffers stay within 64 MB.
    const int64_t chunk_rows = std::min(p.chunk, rows), kb_rows = (chunk_rows + BK - 1) / BK, kb_tokens = (tokens + BK - 1) / BK;
    const int64_t work = p.d_tiles * (p.token_tiles * kb_rows + (chunk_rows + tm - 1) / tm * std::max<int64_t>(kb_tokens, TILE_END));
    const int64_t item = std::max<int64_t>(8, work / (2 * workers));
    const int64_t room = std::max<int64_t>(1, ((int64_t)64 << 20) / (p.token_tiles * tm * (int64_t)dim * 4));
    p.splits = (int)std::min(std::min((kb_rows + item - 1) / item, room), kb_rows);
    // The same for dw, where the table is one chunk.
    p.rows_pad = (chunk_rows + tm - 1) / tm * tm;
    const int64_t room_w = std::max<int64_t>(1, ((int64_t)64 << 20) / (p.rows_pad * dim * 4));
    p.splits_w = chunks > 1 ? 1 : (int)std::min(std::min((kb_tokens + item - 1) / item, room_w), kb_tokens);
    p.off_rho = (size_t)tokens * sizeof(TokenGrad);
    p.off_h = (size_t)up((int64_t)p.off_rho + 4 * (1 + WEIGHT_PARTS), 1024);
    p.off_dh = p.off_h + (size_t)up(tokens * dim * 2, 1024);
    p.off_dw = p.off_dh + (size_t)up((int64_t)p.splits * p.token_tiles * tm * dim * 4, 1024);
    p.off_g = p.off_dw + (p.splits_w > 1 ? (size_t)up(p.splits_w * p.rows_pad * dim * 4, 1024) : 0);
    p.bytes = p.off_g + (size_t)(tokens * p.chunk * 2);
    return p;
}

int check_sizes(int64_t tokens, int64_t rows, int dim) {
    VA_REQUIRE(tokens >= 0 && tokens <= (1 << 24), "tokens must be in 0..16777216, got %lld", (long long)tokens);
    VA_REQUIRE(rows > 0 && rows <= (1 << 28), "rows must be in 1..268435456, got %lld", (long long)rows);
    VA_REQUIRE(dim > 0 && dim <= VA_MAX_DIM && dim % 8 == 0, "dimension must be a multiple of 8 in 8..%d, got %d", VA_MAX_DIM,
               dim);
    VA_REQUIRE((tokens + BM - 1) / BM * ((rows + BM - 1) / BM) <= (1 << 30), "%lld tokens x %lld rows is too large for one call",
               (long long)tokens, (long long)rows);
    return VA_OK;
}

int check_inputs(va_context* ctx, const void* h, int64_t h_stride, const void* table, int64_t table_stride, int64_t tokens,
                 int64_t rows, int dim, float scale) {
    VA_TRY(check_sizes(tokens, rows, dim));
    VA_REQUIRE(h_stride >= dim && h_stride % 8 == 0 && h_stride < ((int64_t)1 << 36),
               "hidden_stride must be a multiple of 8 and at least the dimension %d, got %lld", dim, (long long)h_stride);
    VA_REQUIRE(table_stride >= dim && table_stride % 8 == 0 && table_stride < ((int64_t)1 << 36),
               "table_stride must be a multiple of 8 and at least the dimension %d, got %lld", dim, (long long)table_stride);
    VA_REQUIRE((((uintptr_t)h | (uintptr_t)table) & 15) == 0, "hidden and table must be aligned to 16 bytes");
    // (the kernels work in powers of two)
    VA_REQUIRE(scale > 0.f && scale * LOG2E < INFINITY, "logit_scale must be positive and finite, and below 2^127, got %g", (double)scale);
    return VA_OK;
}

// The caller's workspace, or the context's scratch (which may grow, so never inside a capture).
int workspace_of(va_context* ctx, void* workspace, size_t have, size_t need, void** out) {
    if (workspace) {
        VA_REQUIRE(((uintptr_t)workspace & 127) == 0, "workspace must be aligned to 128 bytes");
        VA_REQUIRE(have >= need, "workspace of %zu bytes is too small: %zu bytes are needed", have, need);
        *out = workspace;
        return VA_OK;
    }
    cudaStreamCaptureStatus status;
    VA_CUDA_TRY(cudaStreamIsCapturing(ctx->stream, &status));
    if (status != cudaStreamCaptureStatusNone)
        return va_set_error(VA_ERR_UNSUPPORTED, "a captured call needs a workspace of its own (%zu bytes)", need);
    return va_workspace(ctx, need, out);
}

// The tile kernels are launched programmatically (see pdl_wait): in a short call their set-up takes as long as their
// work. The small kernels are not: their blocks would wait on the SMs where the tiles are still being worked on, and
// slow them down (64 x 100000 x 768: 48 us instead of 36).
template <auto KERN, typename... Args>
int launch(va_context* ctx, unsigned grid, unsigned block, size_t smem, bool pair, const char* name, Args... args) {
    VA_TRY(va_kernel_once<KERN>(ctx->device, smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = smem ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pair ? 2 : 1;
    VA_CUDA_TRY(cudaLaunchKernelEx(&cfg, KERN, args...));
    return va_check_launch(name);
}

// `items` workers of one or two CTAs, at most one CTA per SM.
template <auto KERN, typename... Args>
int launch_tiles(va_context* ctx, bool pair, int items, const char* name, Args... args) {
    const int grid = pair ? 2 * std::min(ctx->sm_count / 2, items) : std::min(ctx->sm_count, items);
    return launch<KERN>(ctx, (unsigned)grid, THREADS, SMEM, pair, name, args...);
}

template <int MODE>
int launch_scores(va_context* ctx, bool pair, const CUtensorMap& h, const CUtensorMap& w, const CUtensorMap& g,
                  const ScoreWork& work) {
    const int items = work.token_tiles * work.splits;
    const uint64_t limit = wait_limit_ns(ctx->timeout_ms);
    return pair ? launch_tiles<k_xent_scores<MODE, true>>(ctx, true, items, "k_xent_scores", h, w, g, work, ctx->d_error, limit)
                : launch_tiles<k_xent_scores<MODE, false>>(ctx, false, items, "k_xent_scores", h, w, g, work, ctx->d_error, limit);
}

}  // namespace

extern "C" {

int va_softmax_xent_workspace(va_context* ctx, int64_t tokens, int64_t rows, int dim, int backward, size_t* bytes) {
    VA_REQUIRE(ctx && bytes, "ctx and bytes must not be NULL");
    VA_TRY(check_sizes(tokens, rows, dim));
    *bytes = !tokens ? 0 : backward ? plan_backward(ctx->sm_count, tokens, rows, dim).bytes
                                    : plan_forward(ctx->sm_count, tokens, rows).bytes;
    return VA_OK;
}

int va_softmax_xent_forward(va_context* ctx, const uint16_t* hidden, int64_t hidden_stride, const uint16_t* table,
                            int64_t table_stride, const int64_t* labels, int64_t tokens, int64_t rows, int dim,
                            float logit_scale, void* workspace, size_t workspace_bytes, float* loss, float* lse) {
    VA_REQUIRE(ctx && (!tokens || (hidden && table && labels && loss && lse)),
               "ctx, hidden, table, labels, loss and lse must not be NULL");
    VA_TRY(check_inputs(ctx, hidden, hidden_stride, table, table_stride, tokens, rows, dim, logit_scale));
    VA_REQUIRE((((uintptr_t)labels & 7) | (((uintptr_t)loss | (uintptr_t)lse) & 3)) == 0,
               "labels, loss and lse must be aligned to their elements");
    if (!tokens) return VA_OK;
    const VaSpan sh{"hidden", hidden, dim * 2, tokens, hidden_stride * 2}, st{"table", table, dim * 2, rows, table_stride * 2},
        sy{"labels", labels, tokens * 8}, so{"loss", loss, tokens * 4}, se{"lse", lse, tokens * 4};
    VA_TRY(va_refuse_overlap(so, {sh, st, sy, se}));
    VA_TRY(va_refuse_overlap(se, {sh, st, sy}));
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const ForwardPlan p = plan_forward(ctx->sm_count, tokens, rows);
    void* ws;
    VA_TRY(workspace_of(ctx, workspace, workspace_bytes, p.bytes, &ws));
    VA_TRY(va_refuse_overlap({"workspace", workspace, (int64_t)p.bytes}, {sh, st, sy, so, se}));
    CUtensorMap mh, mw;
    VA_TRY(make_map(&mh, hidden, false, dim, tokens, hidden_stride, BK, BM));
    VA_TRY(make_map(&mw, table, false, dim, rows, table_stride, BK, p.pair ? BN / 2 : p.n));
    ScoreWork w{};
    w.n = p.n;
    w.tokens = tokens;
    w.rows = rows;
    w.token_tiles = p.token_tiles;
    w.row_tiles = p.row_tiles;
    w.splits = p.splits;
    w.k_blocks = (dim + BK - 1) / BK;
    w.scale2 = logit_scale * LOG2E;
    w.part = static_cast<float2*>(ws);
    w.stall_tiles = test_stall_tiles();
    w.labels = labels;
    w.label_dot = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.off_dot);
    VA_TRY(launch_scores<FORWARD>(ctx, p.pair, mh, mw, mh, w));
    return launch<k_xent_join>(ctx, (unsigned)((tokens + 3) / 4), 128, 0, false, "k_xent_join", (const float2*)w.part, 2 * p.splits,
                  (int64_t)p.token_tiles * (p.pair ? 2 * BM : BM), (const float*)w.label_dot, labels, tokens, rows, logit_scale, w.scale2,
                  loss, lse);
}

int va_softmax_xent_backward(va_context* ctx, const uint16_t* hidden, int64_t hidden_stride, const uint16_t* table,
                             int64_t table_stride, const int64_t* labels, const float* lse, const float* grad_loss,
                             int64_t tokens, int64_t rows, int dim, float logit_scale, void* workspace,
                             size_t workspace_bytes, uint16_t* grad_hidden, uint16_t* grad_table) {
    VA_REQUIRE(ctx && table && grad_table && (!tokens || (hidden && labels && lse && grad_hidden)),
               "ctx, hidden, table, labels, lse, grad_hidden and grad_table must not be NULL");
    VA_TRY(check_inputs(ctx, hidden, hidden_stride, table, table_stride, tokens, rows, dim, logit_scale));
    VA_REQUIRE((((uintptr_t)grad_hidden | (uintptr_t)grad_table) & 15) == 0,
               "grad_hidden and grad_table must be aligned to 16 bytes");
    VA_REQUIRE(grad_table != table && (!tokens || (grad_hidden != hidden && grad_hidden != table && grad_table != hidden)),
               "grad_hidden and grad_table must not be hidden or table: those are read until the end");
    VA_REQUIRE((((uintptr_t)labels & 7) | (((uintptr_t)lse | (uintptr_t)grad_loss) & 3)) == 0,
               "labels, lse and grad_loss must be aligned to their elements");
    const VaSpan sh{"hidden", hidden, dim * 2, tokens, hidden_stride * 2}, st{"table", table, dim * 2, rows, table_stride * 2},
        sy{"labels", labels, tokens * 8}, se{"lse", lse, tokens * 4}, sg{"grad_loss", grad_loss, tokens * 4},
        gh{"grad_hidden", grad_hidden, tokens * dim * 2}, gt{"grad_table", grad_table, rows * dim * 2};
    VA_TRY(va_refuse_overlap(gh, {sh, st, sy, se, sg, gt}));
    VA_TRY(va_refuse_overlap(gt, {sh, st, sy, se, sg}));
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    if (!tokens) {
        VA_CUDA_TRY(cudaMemsetAsync(grad_table, 0, (size_t)rows * dim * 2, ctx->stream));
        return VA_OK;
    }
    const BackwardPlan p = plan_backward(ctx->sm_count, tokens, rows, dim);
    void* ws;
    VA_TRY(workspace_of(ctx, workspace, workspace_bytes, p.bytes, &ws));
    VA_TRY(va_refuse_overlap({"workspace", workspace, (int64_t)p.bytes}, {sh, st, sy, se, sg, gh, gt}));
    TokenGrad* tok = static_cast<TokenGrad*>(ws);
    float* rho = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.off_rho);
    uint16_t* weighted = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(ws) + p.off_h);
    float* dh = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.off_dh);
    float* dw = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.off_dw);
    uint16_t* g = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(ws) + p.off_g);
    const int parts = tokens > FEW_TOKENS ? (int)std::min<int64_t>(WEIGHT_PARTS, (tokens + 255) / 256) : 0;
    if (parts)
        VA_TRY(launch<k_xent_weights>(ctx, (unsigned)parts, 256, 0, false, "k_xent_weights", labels, grad_loss, tokens, rows, logit_scale,
                      rho + 1));
    VA_TRY(launch<k_xent_tokens>(ctx, (unsigned)((tokens + 3) / 4), 128, 0, false, "k_xent_tokens", hidden, hidden_stride, labels, lse,
                  grad_loss, tokens, rows, dim, logit_scale, (const float*)(rho + 1), parts, tok, rho, weighted));

    const int tm = p.pair ? 2 * BM : BM;
    const int64_t tokens_pad = (int64_t)p.token_tiles * tm;
    CUtensorMap mh, mw, mw64, mh64, mdh, mdw, mdwp;
    VA_TRY(make_map(&mh, hidden, false, dim, tokens, hidden_stride, BK, BM));
    VA_TRY(make_map(&mw, table, false, dim, rows, table_stride, BK, p.pair ? BN / 2 : p.n_scores));
    VA_TRY(make_map(&mh64, weighted, false, dim, tokens, dim, 64, 64));
    VA_TRY(make_map(&mw64, table, false, dim, rows, table_stride, 64, 64));
    VA_TRY(make_map(&mdh, dh, true, dim, p.splits * tokens_pad, dim, 32, 32));
    VA_TRY(make_map(&mdw, grad_table, false, dim, rows, dim, 64, 32));
    mdwp = mdw;
    if (p.splits_w > 1) VA_TRY(make_map(&mdwp, dw, true, dim, p.splits_w * p.rows_pad, dim, 32, 32));
    for (int64_t row0 = 0; row0 < rows; row0 += p.chunk) {
        const int64_t count = std::min(p.chunk, rows - row0);
        CUtensorMap mg_out, mg;
        VA_TRY(make_map(&mg_out, g, false, count, tokens, p.chunk, 64, 32));
        VA_TRY(make_map(&mg, g, false, count, tokens, p.chunk, 64, 64));
        ScoreWork s{};
        s.tokens = tokens;
        s.rows = count;
        s.row0 = row0;
        s.token_tiles = p.token_tiles;
        s.n = p.n_scores;
        s.row_tiles = s.splits = (int)((count + s.n - 1) / s.n);
        s.k_blocks = (dim + BK - 1) / BK;
        s.scale2 = logit_scale * LOG2E;
        s.tok = tok;
        s.stall_tiles = test_stall_tiles();
        VA_TRY(launch_scores<GRADIENT>(ctx, p.pair, mh, mw, mg_out, s));

        GradWork w{};
        w.row0 = row0;
        w.rows = rows;
        w.dim = dim;
        w.tokens = tokens;
        w.tokens_pad = tokens_pad;
        w.token_tiles = p.token_tiles;
        w.row_tiles = (int)((count + tm - 1) / tm);
        w.d_tiles = p.d_tiles;
        w.splits = p.splits;
        w.splits_w = p.splits_w;
        w.rows_pad = p.rows_pad;
        w.rho = rho;
        w.n = p.n;
        w.kb_rows = (int)((count + BK - 1) / BK);
        w.kb_tokens = (int)((tokens + BK - 1) / BK);
        w.first = row0 == 0;
        w.stall_tiles = s.stall_tiles;
        const int items_h = p.token_tiles * p.d_tiles * p.splits, items_w = w.row_tiles * p.d_tiles * p.splits_w;
        const double cost_h = std::max<double>(TILE_END, (double)w.kb_rows / p.splits);
        const double cost_w = std::max<double>(TILE_END, (double)w.kb_tokens / p.splits_w);
        w.long_h = cost_h >= cost_w;
        w.extra = (int)std::lround(std::max(cost_h, cost_w) / std::max(1.0, std::min(cost_h, cost_w)));
        const uint64_t limit = wait_limit_ns(ctx->timeout_ms);
        if (p.pair)
            VA_TRY(launch_tiles<k_xent_grads<true>>(ctx, true, items_h + items_w, "k_xent_grads", mg, mw64, mh64, mdh, mdw, mdwp, w,
                                                    ctx->d_error, limit));
        else
            VA_TRY(launch_tiles<k_xent_grads<false>>(ctx, false, items_h + items_w, "k_xent_grads", mg, mw64, mh64, mdh, mdw, mdwp, w,
                                                     ctx->d_error, limit));
    }
    const auto finish = [&](const float* part, int splits, int64_t pad, int64_t n_rows, const TokenGrad* of, uint16_t* out) {
        const int64_t n4 = n_rows * dim / 4;
        int lanes = 1;
        while (lanes < 16 && splits >= 4 * lanes && n4 * lanes < (int64_t)ctx->sm_count * 512) lanes *= 2;
        const int64_t blocks = (n4 * lanes + 255) / 256;
        return launch<k_xent_finish>(ctx, (unsigned)std::min<int64_t>(blocks, (int64_t)ctx->sm_count * 8), 256, 0, false,
                                     "k_xent_finish", (const float4*)part, splits, lanes, pad * dim / 4, n4, dim / 4, of,
                                     (const float*)rho, (uint2*)out);
    };
    if (p.splits_w > 1) VA_TRY(finish(dw, p.splits_w, p.rows_pad, rows, nullptr, grad_table));
    return finish(dh, p.splits, tokens_pad, tokens, tok, grad_hidden);
}

}  // extern "C"
