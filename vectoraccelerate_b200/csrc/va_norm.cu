// va_norm.cu -- root-mean-square norm with the residual's addition and an int8 output with scales.
//
// Per row of `dim` elements (x, residual and weight of one type, fp32 or bf16):
//   h_j    = x_j + residual_j, rounded to the type when it is bf16 (what residual_out stores)
//   z_j    = h_j * weight_j
//   a      = max |z_j| over the row, or over each group of 32, 64 or 128 columns
//   code_j = rint(127 z_j / a)
//   scale  = a / (127 sqrt(mean(h^2) + eps)),   so that code_j * scale ~ z_j / rms(h)
// The rms cancels from the codes, which are therefore exact: the fp32 quotient decides a code
// except within 2^-14 of a border between two codes (one element in 8,000), where the exact
// remainder does. The sum of squares and the scales are fp32. A row (or group) with
// a < 2^-80 has codes 0 and scale 0. A row whose sum of squares is not finite, and a group whose a is
// not finite, has codes 0 and scale NaN.
//
// The work is one read of x and residual, one write of residual_out and the codes: HBM-bound, with
// ~20 instructions per element to hide. A thread holds one or two vectors of 8 elements of a row in registers between
// the statistics and the codes, so nothing is read twice. Blocks are persistent: while a row is worked on the next one
// comes through cp.async into shared memory, the weights stay in registers, and a row costs one block barrier.
// Measured: 65536 x 4096 bf16 with residual 291 us, 6.5 TB/s; 32768 x 4096 fp32 394 us, 4.4 TB/s; without a residual
// (3 bytes an element) the instructions show: 65536 x 4096 bf16 244 us, 3.3 TB/s.
// Rows that do not start on 16-byte boundaries are copied as the 16-byte pieces that hold them and cut out by shifts;
// results go through shared memory to whole 16-byte (codes: 8-byte) stores, one row later for the codes: 32768 x 4091 fp32
// within 2% of the aligned time, 16384 x 4095 bf16 with residual 140 us (element by element 281, aligned 78). Narrow rows lose by
// it: 400000 x 67 bf16 took 166 us element by element and takes 175 to 184.
#include <algorithm>

#include "va_internal.cuh"

namespace {

// A largest |z| below this counts as zero: fp32 quotients have run out of range by then.
constexpr float SMALLEST = 0x1p-80f;
// A sum of squares below SMALL_SUM may have lost squares to fp32's range (2^-149 each, 2^-41 of a sum above it). An
// epsilon of SMALL_EPS covers that; kernels for a smaller one take the sum again, of elements times 2^100. (A
// variant of their own: in the others the rare case would spill registers.)
constexpr float SMALL_SUM = 0x1p-96f, SMALL_EPS = 0x1p-80f, LIFT = 0x1p100f;

struct NormArgs {
    const void* x;
    const void* residual;
    const void* weight;
    void* residual_out;
    int8_t* codes;
    float* scales;
    int64_t rows, x_stride, residual_stride;
    int dim, group, groups;
    float eps;
};

// Eight elements as loaded: bf16 pairs, or fp32.
template <typename T>
struct Vec {
    uint32_t w[sizeof(T) * 2];
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 2)
            return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        else
            return __uint_as_float(w[i]);
    }
};

// Eight elements from p, `n` of them inside the row (the others read as 0).
template <typename T, bool ALIGNED>
__device__ __forceinline__ Vec<T> load8(const T* p, int n) {
    Vec<T> v;
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 u = n > 0 ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
            v.w[4 * i] = u.x, v.w[4 * i + 1] = u.y, v.w[4 * i + 2] = u.z, v.w[4 * i + 3] = u.w;
        }
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = 2 * i < n ? p[2 * i] : (T)0, hi = 2 * i + 1 < n ? p[2 * i + 1] : (T)0;
            v.w[i] = lo | (hi << 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.w[i] = i < n ? __float_as_uint(p[i]) : 0u;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Vec<T>& v) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(v.w[4 * i], v.w[4 * i + 1], v.w[4 * i + 2], v.w[4 * i + 3]);
}

// The eight elements that start `s` elements (less than 16 bytes) into the 16-byte pieces at p in shared memory.
template <typename T>
__device__ __forceinline__ Vec<T> window8(const uint4* p, int s) {
    constexpr int N = sizeof(T) * 2, MORE = sizeof(T) == 2 ? 1 : 0;  // words; one more where halves are joined
    uint32_t u[N + 4], v[N + MORE + 1];
#pragma unroll
    for (int i = 0; i < N / 4 + 1; ++i) {
        const uint4 q = p[i];
        u[4 * i] = q.x, u[4 * i + 1] = q.y, u[4 * i + 2] = q.z, u[4 * i + 3] = q.w;
    }
    const int words = MORE ? s >> 1 : s;
#pragma unroll
    for (int i = 0; i < N + MORE + 1; ++i) v[i] = words & 2 ? u[i + 2] : u[i];
#pragma unroll
    for (int i = 0; i < N + MORE; ++i) v[i] = words & 1 ? v[i + 1] : v[i];
    Vec<T> out;
    const uint32_t halves = s & 1 ? 0x5432u : 0x3210u;
#pragma unroll
    for (int i = 0; i < N; ++i) out.w[i] = MORE ? __byte_perm(v[i], v[i + MORE], halves) : v[i];
    return out;
}

// Rows in memory that start anywhere: `past` elements after an 8-element boundary of their own. Elements before `head`
// and from `tail` on lie in boundaries shared with neighbouring rows and are stored one by one.
struct Edges {
    int head, tail;
    __device__ __forceinline__ Edges(int past, int dim) {
        head = past ? min(8 - past, dim) : 0;
        tail = head + ((dim - head) & ~7);
    }
    // Which element thread t of the row's first 16 stores, or -1.
    __device__ __forceinline__ int of(int t, int dim) const {
        if (t < 8) return t < head ? t : -1;
        return t < 16 && tail + t - 8 < dim ? tail + t - 8 : -1;
    }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// max(a, |b|), a NaN wins
__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float d;
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Packed bf16 through the mixed-precision fma: a + b as fp32, and a b + c exactly as fp32 fma of the two values.
// (As fast as an fp32 fma, where unpacking by shift or mask runs at half that rate.)
template <int HALF>
__device__ __forceinline__ float fma_half(uint32_t a, uint32_t b, float c) {
    float d;
    if constexpr (HALF == 0)
        asm("{\n\t.reg .b16 al, ah, bl, bh;\n\tmov.b32 {al, ah}, %1;\n\tmov.b32 {bl, bh}, %2;\n\tfma.rn.f32.bf16 %0, al, bl, %3;\n\t}"
            : "=f"(d)
            : "r"(a), "r"(b), "f"(c));
    else
        asm("{\n\t.reg .b16 al, ah, bl, bh;\n\tmov.b32 {al, ah}, %1;\n\tmov.b32 {bl, bh}, %2;\n\tfma.rn.f32.bf16 %0, ah, bh, %3;\n\t}"
            : "=f"(d)
            : "r"(a), "r"(b), "f"(c));
    return d;
}

// x + r, rounded to the type.
template <typename T>
__device__ __forceinline__ Vec<T> add8(const Vec<T>& x, const Vec<T>& r) {
    Vec<T> h;
    if constexpr (sizeof(T) == 2) {
        constexpr uint32_t ONE = 0x3F803F80u;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            h.w[k] = pack_bf16(fma_half<0>(x.w[k], ONE, fma_half<0>(r.w[k], ONE, 0.f)),
                               fma_half<1>(x.w[k], ONE, fma_half<1>(r.w[k], ONE, 0.f)));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) h.w[k] = __float_as_uint(x[k] + r[k]);
    }
    return h;
}

// z = h w (exact for bf16) and the sum of squares of h.
template <typename T>
__device__ __forceinline__ void products(const Vec<T>& h, const Vec<T>& w, float (&z)[8], float& sum) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if constexpr (sizeof(T) == 2) {
            z[k] = k & 1 ? fma_half<1>(h.w[k >> 1], w.w[k >> 1], 0.f) : fma_half<0>(h.w[k >> 1], w.w[k >> 1], 0.f);
            sum = k & 1 ? fma_half<1>(h.w[k >> 1], h.w[k >> 1], sum) : fma_half<0>(h.w[k >> 1], h.w[k >> 1], sum);
        } else {
            z[k] = h[k] * w[k];
            sum = fmaf(h[k], h[k], sum);
        }
    }
}

// The largest |z| so far, exactly: z = hi + lo with hi = fl(z). Rounding is monotonic, so hi decides
// and lo only breaks ties of hi. Products of two bf16 values fit fp32: lo stays 0. A NaN stays in hi (and
// is then reported through the scale).
template <typename T>
struct Top {
    float hi = 0.f, lo = 0.f;
    __device__ __forceinline__ void take(float h, float l) {
        if constexpr (sizeof(T) == 2) {
            hi = max_abs_nan(hi, h);
        } else {
            const bool more = hi == hi && (!(h <= hi) || (h == hi && l > lo));  // a NaN wins from either side
            lo = more ? l : lo;
            hi = more ? h : hi;
        }
    }
    // Of a thread's eight elements: the largest hi first, then lo among the (nearly always one) that have it.
    __device__ __forceinline__ void of(const Vec<T>& h, const Vec<T>& w, const float (&z)[8]) {
#pragma unroll
        for (int k = 0; k < 8; ++k) hi = max_abs_nan(hi, z[k]);
        if constexpr (sizeof(T) == 4) {
            lo = -INFINITY;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (fabsf(z[k]) == hi) lo = fmaxf(lo, copysignf(1.f, z[k]) * fmaf(h[k], w[k], -z[k]));
        }
    }
    template <int WIDTH>
    __device__ __forceinline__ void lanes() {
        if constexpr (WIDTH == 32) {
            // non-negative floats (and a NaN above them) order like their bits, negative ones against them
            const uint32_t own = __float_as_uint(hi), top = __reduce_max_sync(0xFFFFFFFFu, own);
            if constexpr (sizeof(T) == 4) {
                const auto ordered = [](int b) { return b ^ ((b >> 31) & 0x7FFFFFFF); };
                const int low = __reduce_max_sync(0xFFFFFFFFu, own == top ? ordered(__float_as_int(lo)) : (int)0x80000000);
                lo = __int_as_float(ordered(low));
            }
            hi = __uint_as_float(top);
        } else {
#pragma unroll
            for (int o = 1; o < WIDTH; o <<= 1) {
                const float h = __shfl_xor_sync(0xFFFFFFFFu, hi, o);
                const float l = sizeof(T) == 2 ? 0.f : __shfl_xor_sync(0xFFFFFFFFu, lo, o);
                take(h, l);
            }
        }
    }
    __device__ __forceinline__ void lanes(int width) {
        if (width == 4)
            lanes<4>();
        else if (width == 8)
            lanes<8>();
        else
            lanes<16>();
    }
};

// rint(127 z / a) of eight elements, packed. t = z (127 / a) in fp32 is within 127 * 3 * 2^-24 < 2^-15 of the
// quotient; adding 1.5 * 2^23 rounds it (to even) into the low byte. Where some t is within 2^-14 of the border
// b between two codes, the sign of 127 z - b a decides: for bf16 both products are exact in fp32 (7 + 16 and 8 + 16
// bits); for fp32 their rounding errors and the low parts are added (48 bits).
template <typename T>
__device__ __forceinline__ uint2 codes_of(const Vec<T>& h, const Vec<T>& w, const float (&z)[8], const Top<T>& a) {
    uint32_t m[8];
    constexpr float SHIFT = 12582912.f;
    constexpr float NEAR = 0.5f - 0x1p-14f;
    const float inv = 127.f / a.hi;
    float off = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float t = z[k] * inv, r = t + SHIFT;
        m[k] = __float_as_uint(r);
        off = fmaxf(off, fabsf(t - (r - SHIFT)));
    }
    if (off > NEAR) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float t = z[k] * inv, r = __uint_as_float(m[k]) - SHIFT, d = t - r;
            if (fabsf(d) > NEAR) {
                const float b = r + copysignf(0.5f, d), p = b * a.hi, q = 127.f * z[k];
                float diff = q - p;
                if constexpr (sizeof(T) == 4)
                    diff += (fmaf(127.f, z[k], -q) - fmaf(b, a.hi, -p)) + (127.f * fmaf(h[k], w[k], -z[k]) - b * a.lo);
                const float past = copysignf(diff, 1.f) == 0.f ? ((m[k] & 1u) ? 1.f : -1.f) : (d > 0.f ? diff : -diff);
                if (past > 0.f) m[k] += d > 0.f ? 1u : 0xFFFFFFFFu;
            }
        }
    }
    uint2 p;
    p.x = __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
    p.y = __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410);
    return p;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// As cp_async16, of the first `bytes`; the rest becomes zero.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A block works on one row at a time with TPR threads of NV vectors (8 elements) each. (Narrow rows do not share a
// block: with rows, addresses and barriers of a warp's own, 200000 x 128 bf16 took 72 us instead of 68.) Two vectors
// share the reductions' cost (bf16, 65536 x 4096: 316 us, with one 390 us; fp32, at 128 registers, 32768 x 4096: 395 us, with
// one at 80 475 us).
template <typename T, bool ALIGNED, int TPR, int NV>
struct Plan {
    static constexpr int HALVES = sizeof(T) / 2;  // 16-byte pieces of a vector
    // Rows in work or on their way. (Three: 65536 x 4096 bf16 with residual 338 us instead of 293.)
    static constexpr int STAGES = 2;
    // Shared memory. ALIGNED: [stage][x, residual][vector][piece][thread] of 16 bytes. Else rows as they lie in
    // memory, [stage][x, residual][piece], then [2][piece] of residual_out and [2][vector] of codes (8 bytes).
    static constexpr int PIECES = TPR * NV * HALVES + 1;  // of a row that starts inside its first
    static constexpr int CODES = TPR * NV + 1;
    static constexpr int OUT = STAGES * 2 * PIECES;
    static constexpr int BYTES = ALIGNED ? STAGES * 2 * NV * HALVES * TPR * 16 : (OUT + 2 * PIECES) * 16 + 2 * CODES * 8;
    // Blocks per SM: 768 threads of up to 80 registers, or 512 of 128 where two fp32 vectors take them, if their
    // shared memory (with 1 KB of the system's and the static part) fits the SM's 228 KB: all blocks have to run at once.
    static constexpr int WANTED = (sizeof(T) * NV == 8 ? 512 : 768) / TPR;
    static constexpr int FIT = 228 * 1024 / (BYTES + 1024 + TPR / 32 * 32);
    static constexpr int BLOCKS = WANTED < FIT ? WANTED : FIT;
};

// A row's residual_out and codes from shared memory to any address: whole 16 (codes: 8) bytes and edges. A thread's
// vectors are t, t + TPR, ...
template <typename T, int NV, int TPR>
__device__ __forceinline__ void put_row(T* out, int dim, const uint4* from, int t) {
    constexpr int A = 16 / sizeof(T), HALVES = sizeof(T) / 2;
    const int m = (int)((uintptr_t)out / sizeof(T)) & (A - 1);
    const Edges edge(m, dim);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = t + i * TPR, at = v * 8 - m;
        if (at >= edge.head && at < edge.tail)
            store8<T>(out + at, window8<T>(from + v * HALVES - (m ? 1 : 0), (A - m) & (A - 1)));
    }
    const int e = edge.of(t, dim);
    if (e >= 0) out[e] = reinterpret_cast<const T*>(from)[e];
}

template <int NV, int TPR>
__device__ __forceinline__ void put_codes(int8_t* out, int dim, const uint2* from, int t) {
    const int m = (int)((uintptr_t)out & 7), s = (8 - m) & 7;
    const Edges edge(m, dim);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = t + i * TPR, at = v * 8 - m;
        if (at >= edge.head && at < edge.tail) {
            const uint2 p = from[v - (m ? 1 : 0)], q = from[v - (m ? 1 : 0) + 1];
            const uint32_t u0 = s & 4 ? p.y : p.x, u1 = s & 4 ? q.x : p.y, u2 = s & 4 ? q.y : q.x;
            *reinterpret_cast<uint2*>(out + at) = make_uint2(__funnelshift_r(u0, u1, 8 * (s & 3)), __funnelshift_r(u1, u2, 8 * (s & 3)));
        }
    }
    const int e = edge.of(t, dim);
    if (e >= 0) out[e] = reinterpret_cast<const int8_t*>(from)[e];
}

// Vector i of thread t is at (i * TPR + t) * 8.
template <typename T, bool ALIGNED, int TPR, int NV, bool SMALL>
__global__ void __launch_bounds__(TPR, Plan<T, ALIGNED, TPR, NV>::BLOCKS) k_rms_norm_int8(NormArgs a) {
    using P = Plan<T, ALIGNED, TPR, NV>;
    constexpr int WARPS = TPR / 32, STAGES = P::STAGES, HALVES = P::HALVES;
    constexpr int A = 16 / sizeof(T), ES = sizeof(T);  // elements of a piece
    extern __shared__ uint4 s_in[];
    __shared__ float4 s_part[2][WARPS];  // (sum, hi, lo, -) of each warp
    __shared__ float s_again[SMALL ? WARPS : 1];  // a small row's sum
    const int t = threadIdx.x, j0 = t * 8;
    Vec<T> w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        w[i] = load8<T, ALIGNED>(static_cast<const T*>(a.weight) + j0 + i * TPR * 8, a.dim - j0 - i * TPR * 8);
    const uint32_t step = gridDim.x, rows = (uint32_t)a.rows;  // (below 2^31: a row index plus step fits)
    uint32_t row = blockIdx.x, ahead = row;
    const int lead = ALIGNED ? j0 : 0;
    const T* px = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride + lead;
    const T* pr = a.residual ? static_cast<const T*>(a.residual) + (int64_t)row * a.residual_stride + lead : nullptr;
    const auto in_row = [&](int stage, int which) { return s_in + (stage * 2 + which) * P::PIECES; };
    const auto out_row = [&](int turn) { return s_in + P::OUT + turn * P::PIECES; };
    const auto code_row = [&](int turn) { return reinterpret_cast<uint2*>(s_in + P::OUT + 2 * P::PIECES) + turn * P::CODES; };
    const auto barrier = [&] {
        if constexpr (WARPS > 1)
            __syncthreads();
        else
            __syncwarp();
    };
    // Elements between a 16-byte boundary and the start of a row.
    const auto past = [](const void* p, uint32_t row, int64_t stride) {
        return (int)(((uint32_t)((uintptr_t)p / ES) + row * (uint32_t)stride) & (A - 1));
    };
    // The pieces of a row, from the boundary before it (which its allocation holds) to its last element.
    const auto fetch_pieces = [&](uint4* to, const T* from) {
        const int before = (int)((uintptr_t)from / ES) & (A - 1), end = (a.dim + before) * ES;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(from - before);
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
#pragma unroll
        for (int i = 0; i < NV * HALVES; ++i) {
            const int at = (t + i * TPR) * 16;
            if (at < end) cp_async16(dst + at, src + at, min(16, end - at));
        }
        constexpr int LAST = TPR * NV * HALVES * 16;
        if (t == 0 && LAST < end) cp_async16(dst + LAST, src + LAST, end - LAST);
    };
    // Row `ahead` into a stage; px and pr point at it and move on.
    const auto fetch = [&](int stage) {
        if (ahead < rows) {
            if constexpr (ALIGNED) {
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(s_in + stage * 2 * NV * HALVES * TPR + t);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (j0 + i * TPR * 8 >= a.dim) continue;
#pragma unroll
                    for (int p = 0; p < HALVES; ++p)
                        cp_async16(dst + (i * HALVES + p) * TPR * 16, reinterpret_cast<const uint4*>(px + i * TPR * 8) + p);
                    if (pr) {
#pragma unroll
                        for (int p = 0; p < HALVES; ++p)
                            cp_async16(dst + ((NV + i) * HALVES + p) * TPR * 16,
                                       reinterpret_cast<const uint4*>(pr + i * TPR * 8) + p);
                    }
                }
            } else {
                fetch_pieces(in_row(stage, 0), px);
                if (pr) fetch_pieces(in_row(stage, 1), pr);
            }
        }
        cp_async_commit();
        ahead += step;
        px += step * a.x_stride;
        if (pr) pr += step * a.residual_stride;
    };
    // A vector of the current row from its stage.
    const auto take = [&](int stage, int which, int i, int before) {
        Vec<T> v;
        if constexpr (ALIGNED) {
            const uint4* from = s_in + ((stage * 2 + which) * NV + i) * HALVES * TPR + t;
#pragma unroll
            for (int p = 0; p < HALVES; ++p) {
                const uint4 u = from[p * TPR];
                v.w[4 * p] = u.x, v.w[4 * p + 1] = u.y, v.w[4 * p + 2] = u.z, v.w[4 * p + 3] = u.w;
            }
        } else {
            v = window8<T>(in_row(stage, which) + (t + i * TPR) * HALVES, before);
            const int n = a.dim - j0 - i * TPR * 8;
            if (n < 8) {  // (what lies behind the row is not its)
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) * 2; ++k) {
                    if constexpr (ES == 2)
                        v.w[k] = 2 * k + 1 < n ? v.w[k] : 2 * k < n ? v.w[k] & 0xFFFFu : 0u;
                    else
                        v.w[k] = k < n ? v.w[k] : 0u;
                }
            }
        }
        return v;
    };
    for (int s = 0; s < STAGES - 1; ++s) fetch(s);
    if constexpr (!ALIGNED) {
        cp_async_wait<STAGES - 2>();
        barrier();
    }
    int stage = 0, turn = 0;
    // The current row's residual_out and codes.
    T* out = static_cast<T*>(a.residual_out) + (int64_t)row * a.dim + lead;
    int8_t* codes = a.codes + (int64_t)row * a.dim + lead;
    float* scales = a.scales + (int64_t)row * a.groups;
    const int64_t out_step = (int64_t)step * a.dim, scale_step = (int64_t)step * a.groups;
    const float mean = 1.f / (float)a.dim;
    for (; row < rows; row += step, turn ^= 1) {
        // (residual_out may be x's or residual's own rows: a row is stored only after its loads.)
        fetch(stage == 0 ? STAGES - 1 : stage - 1);
        if constexpr (ALIGNED) cp_async_wait<STAGES - 1>();
        const int before_x = past(a.x, row, a.x_stride), before_r = past(a.residual, row, a.residual_stride);
        Vec<T> h[NV] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (j0 + i * TPR * 8 < a.dim) {
                h[i] = take(stage, 0, i, before_x);
                if (a.residual) h[i] = add8<T>(h[i], take(stage, 1, i, before_r));
            }
        if (a.residual_out) {
            T* to = ALIGNED ? out : reinterpret_cast<T*>(out_row(turn)) + j0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (j0 + i * TPR * 8 < a.dim) store8<T>(to + i * TPR * 8, h[i]);
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        float sum = 0.f, z[NV][8];
        Top<T> top[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            products<T>(h[i], w[i], z[i], sum);
            top[i].of(h[i], w[i], z[i]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (a.group) {
#pragma unroll
            for (int i = 0; i < NV; ++i) top[i].lanes(a.group / 8);
        } else {
#pragma unroll
            for (int i = 1; i < NV; ++i) top[0].take(top[i].hi, top[i].lo);
            top[0].template lanes<32>();
        }
        // (Two sets of everything that threads exchange, in turn: one barrier per row.)
        if constexpr (!ALIGNED) cp_async_wait<STAGES - 2>();  // the next row is there behind the barrier
        if constexpr (WARPS > 1) {
            // Lane i takes warp i's part, then the lanes add up.
            if ((t & 31) == 0) s_part[turn][t >> 5] = make_float4(sum, top[0].hi, top[0].lo, 0.f);
            barrier();
            const float4 p = s_part[turn][t & (WARPS - 1)];
            sum = p.x;
#pragma unroll
            for (int o = 1; o < WARPS; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (!a.group) {
                top[0].hi = p.y;
                top[0].lo = p.z;
                top[0].template lanes<32>();  // (each warp's part is there 32 / WARPS times)
            }
        } else if constexpr (!ALIGNED) {
            barrier();
        }
        if constexpr (!ALIGNED) {
            if (a.residual_out) put_row<T, NV, TPR>(out, a.dim, out_row(turn), t);
            // the row before's (a block's first row is below step)
            if (row >= step) put_codes<NV, TPR>(codes - out_step, a.dim, code_row(turn ^ 1), t);
        }
        if (!a.group) {
#pragma unroll
            for (int i = 1; i < NV; ++i) top[i] = top[0];
        }
        // (All threads of the row have the same sum; its sign then says which one it is.)
        if (SMALL && sum < SMALL_SUM) {
            float again = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) again = fmaf(h[i][k] * LIFT, h[i][k] * LIFT, again);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) again += __shfl_xor_sync(0xFFFFFFFFu, again, o);
            if constexpr (WARPS > 1) {
                // (the next row's barrier lies between these reads and the next writes)
                if ((t & 31) == 0) s_again[t >> 5] = again;
                barrier();
                again = s_again[t & (WARPS - 1)];
#pragma unroll
                for (int o = 1; o < WARPS; o <<= 1) again += __shfl_xor_sync(0xFFFFFFFFu, again, o);
            }
            sum = -again;
        }
        uint2* to = ALIGNED ? reinterpret_cast<uint2*>(codes) : code_row(turn) + t;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = j0 + i * TPR * 8;
            if (j >= a.dim) continue;
            const bool ok = sum < INFINITY && top[i].hi < INFINITY;  // false for NaN too
            if (a.group ? (j & (a.group - 1)) == 0 : j == 0) {
                const bool lifted = SMALL && signbit(sum);
                const float per = rsqrtf(lifted ? a.eps * LIFT * LIFT - sum * mean : sum * mean + a.eps) * (1.f / 127.f);
                // (LIFT in two steps: hi * per alone may leave fp32's range at either end)
                const float scale = lifted ? top[i].hi * 0x1p40f * per * (LIFT * 0x1p-40f) : top[i].hi * per;
                scales[a.group ? j / a.group : 0] = !ok ? __int_as_float(0x7FC00000) : top[i].hi >= SMALLEST ? scale : 0.f;
            }
            uint2 packed = make_uint2(0u, 0u);
            if (ok && top[i].hi >= SMALLEST) packed = codes_of<T>(h[i], w[i], z[i], top[i]);
            to[i * TPR] = packed;
        }
        out += out_step;
        codes += out_step;
        scales += scale_step;
    }
    if constexpr (!ALIGNED) {
        barrier();
        put_codes<NV, TPR>(codes - out_step, a.dim, code_row(turn ^ 1), t);
    }
}

template <typename T, bool ALIGNED, int TPR, int NV, bool SMALL>
int launch_rows(va_context* ctx, const NormArgs& a) {
    using P = Plan<T, ALIGNED, TPR, NV>;
    constexpr auto kern = k_rms_norm_int8<T, ALIGNED, TPR, NV, SMALL>;
    VA_TRY(va_kernel_once<kern>(ctx->device, P::BYTES));
    const int64_t grid = std::min<int64_t>(a.rows, (int64_t)ctx->sm_count * P::BLOCKS);
    kern<<<(unsigned)grid, TPR, P::BYTES, ctx->stream>>>(a);
    return va_check_launch("k_rms_norm_int8");
}

template <typename T, bool ALIGNED, bool SMALL>
int launch_width(va_context* ctx, const NormArgs& a) {
    if (a.dim <= 256) return launch_rows<T, ALIGNED, 32, 1, SMALL>(ctx, a);
    if (a.dim <= 512) return launch_rows<T, ALIGNED, 32, 2, SMALL>(ctx, a);
    if (a.dim <= 1024) return launch_rows<T, ALIGNED, 64, 2, SMALL>(ctx, a);
    if (a.dim <= 2048) return launch_rows<T, ALIGNED, 128, 2, SMALL>(ctx, a);
    return launch_rows<T, ALIGNED, 256, 2, SMALL>(ctx, a);
}

template <typename T, bool ALIGNED>
int launch_norm(va_context* ctx, const NormArgs& a) {
    return a.eps < SMALL_EPS ? launch_width<T, ALIGNED, true>(ctx, a) : launch_width<T, ALIGNED, false>(ctx, a);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" {

int va_rms_norm_int8(va_context* ctx, const void* x, const void* residual, const void* weight, int64_t rows, int dim,
                     int dtype, int64_t x_stride, int64_t residual_stride, float eps, int group, void* residual_out,
                     int8_t* codes, float* scales) {
    VA_REQUIRE(ctx && (!rows || (x && weight && codes && scales)), "ctx, x, weight, codes and scales must not be NULL");
    VA_REQUIRE(rows >= 0 && rows <= 0x7FFFFFFF, "rows must be in 0..2147483647, got %lld", (long long)rows);
    VA_REQUIRE(dim > 0 && dim <= VA_MAX_DIM, "dimension must be in 1..%d, got %d", VA_MAX_DIM, dim);
    VA_REQUIRE(dtype == VA_DTYPE_F32 || dtype == VA_DTYPE_BF16, "dtype must be VA_DTYPE_F32 or VA_DTYPE_BF16, got %d",
               dtype);
    VA_REQUIRE(x_stride >= dim, "x_stride must be at least the dimension %d, got %lld", dim, (long long)x_stride);
    VA_REQUIRE(!residual || residual_stride >= dim, "residual_stride must be at least the dimension %d, got %lld", dim,
               (long long)residual_stride);
    VA_REQUIRE(residual || !residual_out, "residual_out needs a residual");
    VA_REQUIRE(!residual_out || ((residual_out != x || x_stride == dim) &&
                                 (residual_out != residual || residual_stride == dim)),
               "residual_out in place needs contiguous rows (stride = dimension %d)", dim);
    VA_REQUIRE(eps >= 0.f && eps < INFINITY, "epsilon must be finite and not negative, got %g", (double)eps);
    VA_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128, "group must be 0 (the row), 32, 64 or 128, got %d",
               group);
    const size_t es = dtype == VA_DTYPE_BF16 ? 2 : 4;
    VA_REQUIRE(((uintptr_t)x % es | (uintptr_t)residual % es | (uintptr_t)weight % es | (uintptr_t)residual_out % es |
                (uintptr_t)scales % 4) == 0,
               "x, residual, weight, residual_out and scales must be aligned to their elements");
    if (!rows) return VA_OK;
    {
        const int64_t n = rows * dim, e = (int64_t)es, groups = group ? (dim + group - 1) / group : 1;
        const VaSpan sx{"x", residual_out == x ? nullptr : x, dim * e, rows, x_stride * e};
        const VaSpan sr{"residual", residual_out == residual ? nullptr : residual, dim * e, rows, residual_stride * e};
        const VaSpan sw{"weight", weight, dim * e}, so{"residual_out", residual_out, n * e}, sc{"codes", codes, n},
            ss{"scales", scales, rows * groups * 4};
        VA_TRY(va_refuse_overlap(so, {sx, sr, sw, sc, ss}));
        VA_TRY(va_refuse_overlap(sc, {sx, sr, sw, ss}));
        VA_TRY(va_refuse_overlap(ss, {sx, sr, sw}));
    }
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const NormArgs a{x,    residual, weight,   residual_out,    codes, scales,
                     rows, x_stride, residual_stride, dim, group, group ? (dim + group - 1) / group : 1, eps};
    // 16-byte accesses when every row starts on a 16-byte boundary and holds whole vectors.
    const bool wide = dim % 8 == 0 && aligned16(x) && aligned16(weight) && x_stride * es % 16 == 0 &&
                      (!residual || (aligned16(residual) && residual_stride * es % 16 == 0)) &&
                      (!residual_out || aligned16(residual_out)) && ((uintptr_t)codes & 7) == 0;
    if (dtype == VA_DTYPE_BF16)
        return wide ? launch_norm<uint16_t, true>(ctx, a) : launch_norm<uint16_t, false>(ctx, a);
    return wide ? launch_norm<float, true>(ctx, a) : launch_norm<float, false>(ctx, a);
}

}  // extern "C"
