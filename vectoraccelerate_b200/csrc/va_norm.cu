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
// the statistics and the codes, so nothing is read twice. Blocks are persistent: each thread's vectors of
// the next rows come through cp.async into shared memory of its own (no barrier), the weights stay in
// registers, and a row costs one block barrier. Measured: 65536 x 4096 bf16 with residual 310 us, 6.0 TB/s; without a
// residual (3 bytes an element) the instructions show: 16384 x 4096 70 us, 2.9 TB/s. Rows without 16-byte alignment are
// read and written element by element, at a quarter to a half of that rate.
#include <algorithm>

#include "va_internal.cuh"

namespace {

// A largest |z| below this counts as zero: fp32 squares and quotients have run out of range by then.
constexpr float SMALLEST = 0x1p-80f;

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

// Eight elements from p, `n` of them inside the row (the others read as 0). W is the widest access in bytes
// that every row start allows: 16, or the element's size.
template <typename T, int W>
__device__ __forceinline__ Vec<T> load8(const T* p, int n) {
    Vec<T> v;
    if constexpr (W == 16) {
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

template <typename T, int W>
__device__ __forceinline__ void store8(T* p, int n, const Vec<T>& v) {
    if constexpr (W == 16) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            reinterpret_cast<uint4*>(p)[i] = make_uint4(v.w[4 * i], v.w[4 * i + 1], v.w[4 * i + 2], v.w[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 2)
                    p[i] = (T)(i & 1 ? v.w[i >> 1] >> 16 : v.w[i >> 1]);
                else
                    p[i] = __uint_as_float(v.w[i]);
            }
    }
}

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
            const bool more = !(h <= hi) || (h == hi && l > lo);
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
        if constexpr (sizeof(T) == 2 && WIDTH == 32) {
            // non-negative floats (and a NaN above them) order like their bits
            hi = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(hi)));
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

constexpr int STAGES = 3;  // rows per thread in work or on their way (16-byte accesses only)

// Threads of a block for rows of TPR threads: narrow rows share a block of 128.
constexpr int threads_of(int tpr) { return tpr < 128 ? 128 : tpr; }
// Vectors of 8 elements per thread: two share the reductions' cost (bf16, 65536 x 4096: 316 us, with one 390 us);
// two of fp32 overflow the registers (10007 x 1000: 31 us, with one 25 us).
template <typename T>
constexpr int vectors_of() { return sizeof(T) == 2 ? 2 : 1; }
// Blocks per SM: 768 threads of up to 80 registers, or 1024 of 64.
template <typename T>
constexpr int blocks_of(int tpr) { return (vectors_of<T>() == 2 ? 768 : 1024) / threads_of(tpr); }

// TPR threads per row; vector i of thread t is at (i * TPR + t) * 8.
template <typename T, int W, int TPR>
__global__ void __launch_bounds__(threads_of(TPR), blocks_of<T>(TPR)) k_rms_norm_int8(NormArgs a) {
    constexpr int THREADS = threads_of(TPR), ROWS = THREADS / TPR, WARPS = TPR / 32, NV = vectors_of<T>();
    constexpr int HALVES = sizeof(T) / 2;  // 16-byte pieces of a vector
    extern __shared__ uint4 s_in[];        // [stage][x, residual][vector][piece][thread]
    __shared__ float4 s_part[2][ROWS][WARPS];  // (sum, hi, lo, -) of each warp
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, j0 = t * 8;
    Vec<T> w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load8<T, W>(static_cast<const T*>(a.weight) + j0 + i * TPR * 8, a.dim - j0 - i * TPR * 8);
    const int64_t step = (int64_t)gridDim.x * ROWS;
    // Every thread of a block makes the same number of turns (barriers); a slot without a row works on zeros.
    int64_t row = (int64_t)blockIdx.x * ROWS + slot, ahead = row;
    int64_t turns = row - slot < a.rows ? (a.rows - (row - slot) + step - 1) / step : 0;
    const T* px = static_cast<const T*>(a.x) + row * a.x_stride + j0;
    const T* pr = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride + j0 : nullptr;
    // Row `ahead` into a stage; px and pr point at it and move on.
    const auto fetch = [&](int stage) {
        if constexpr (W == 16) {
            if (ahead < a.rows) {
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(s_in + stage * 2 * NV * HALVES * THREADS + threadIdx.x);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (j0 + i * TPR * 8 >= a.dim) continue;
#pragma unroll
                    for (int p = 0; p < HALVES; ++p)
                        cp_async16(dst + (i * HALVES + p) * THREADS * 16, reinterpret_cast<const uint4*>(px + i * TPR * 8) + p);
                    if (pr) {
#pragma unroll
                        for (int p = 0; p < HALVES; ++p)
                            cp_async16(dst + ((NV + i) * HALVES + p) * THREADS * 16,
                                       reinterpret_cast<const uint4*>(pr + i * TPR * 8) + p);
                    }
                }
            }
            cp_async_commit();
            ahead += step;
            px += step * a.x_stride;
            if (pr) pr += step * a.residual_stride;
        }
    };
    // A vector of the current row: from its stage, or from memory where rows have no 16-byte alignment.
    const auto take = [&](int stage, int which, int i) {
        if constexpr (W == 16) {
            Vec<T> v;
            const uint4* from = s_in + ((stage * 2 + which) * NV + i) * HALVES * THREADS + threadIdx.x;
#pragma unroll
            for (int p = 0; p < HALVES; ++p) {
                const uint4 u = from[p * THREADS];
                v.w[4 * p] = u.x, v.w[4 * p + 1] = u.y, v.w[4 * p + 2] = u.z, v.w[4 * p + 3] = u.w;
            }
            return v;
        } else {
            return load8<T, W>((which ? pr : px) + i * TPR * 8, a.dim - j0 - i * TPR * 8);
        }
    };
    for (int s = 0; s < STAGES - 1; ++s) fetch(s);
    int stage = 0, turn = 0;
    const float mean = 1.f / (float)a.dim;
    for (; turns > 0; --turns, turn ^= 1) {
        // (residual_out may be x's or residual's own rows: a row is stored only after its loads.)
        fetch(stage == 0 ? STAGES - 1 : stage - 1);
        if constexpr (W == 16) cp_async_wait<STAGES - 1>();
        const bool live = row < a.rows;
        Vec<T> h[NV] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live && j0 + i * TPR * 8 < a.dim) {
                h[i] = take(stage, 0, i);
                if (a.residual) h[i] = add8<T>(h[i], take(stage, 1, i));
            }
        if (a.residual_out && live) {
            T* out = static_cast<T*>(a.residual_out) + row * a.dim + j0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (j0 + i * TPR * 8 < a.dim) store8<T, W>(out + i * TPR * 8, a.dim - j0 - i * TPR * 8, h[i]);
        }
        if constexpr (W != 16) {
            px += step * a.x_stride;
            if (pr) pr += step * a.residual_stride;
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
        if constexpr (WARPS > 1) {
            // Two sets of slots in turn: one barrier per row. Lane i takes warp i's part, then the lanes add up.
            if ((t & 31) == 0) s_part[turn][slot][t >> 5] = make_float4(sum, top[0].hi, top[0].lo, 0.f);
            __syncthreads();
            const float4 p = s_part[turn][slot][t & (WARPS - 1)];
            sum = p.x;
#pragma unroll
            for (int o = 1; o < WARPS; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (!a.group) {
                top[0].hi = p.y;
                top[0].lo = p.z;
                top[0].template lanes<WARPS>();
            }
        }
        if (!a.group) {
#pragma unroll
            for (int i = 1; i < NV; ++i) top[i] = top[0];
        }
        if (live) {
            int8_t* codes = a.codes + row * a.dim + j0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = j0 + i * TPR * 8;
                if (j >= a.dim) continue;
                const bool ok = sum < INFINITY && top[i].hi < INFINITY;  // false for NaN too
                if (a.group ? (j & (a.group - 1)) == 0 : j == 0) {
                    const float per = rsqrtf(sum * mean + a.eps) * (1.f / 127.f);
                    a.scales[row * a.groups + (a.group ? j / a.group : 0)] =
                        !ok ? __int_as_float(0x7FC00000) : top[i].hi >= SMALLEST ? top[i].hi * per : 0.f;
                }
                uint2 packed = make_uint2(0u, 0u);
                if (ok && top[i].hi >= SMALLEST) packed = codes_of<T>(h[i], w[i], z[i], top[i]);
                int8_t* to = codes + i * TPR * 8;
                if constexpr (W == 16) {
                    *reinterpret_cast<uint2*>(to) = packed;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (j + k < a.dim) to[k] = (int8_t)((k < 4 ? packed.x : packed.y) >> (8 * (k & 3)));
                }
            }
        }
        row += step;
    }
}

template <typename T, int W, int TPR>
int launch_rows(va_context* ctx, const NormArgs& a) {
    constexpr int THREADS = threads_of(TPR), ROWS = THREADS / TPR;
    constexpr size_t SMEM = W == 16 ? (size_t)STAGES * 2 * vectors_of<T>() * (sizeof(T) / 2) * THREADS * 16 : 0;
    constexpr auto kern = k_rms_norm_int8<T, W, TPR>;
    VA_TRY(va_kernel_once<kern>(ctx->device, SMEM));
    const int64_t grid = std::min<int64_t>((a.rows + ROWS - 1) / ROWS, (int64_t)ctx->sm_count * blocks_of<T>(TPR));
    kern<<<(unsigned)grid, THREADS, SMEM, ctx->stream>>>(a);
    return va_check_launch("k_rms_norm_int8");
}

template <typename T, int W>
int launch_norm(va_context* ctx, const NormArgs& a) {
    constexpr int PER = 8 * vectors_of<T>();  // elements of a thread
    if (a.dim <= 32 * PER) return launch_rows<T, W, 32>(ctx, a);
    if (a.dim <= 64 * PER) return launch_rows<T, W, 64>(ctx, a);
    if (a.dim <= 128 * PER) return launch_rows<T, W, 128>(ctx, a);
    if (a.dim <= 256 * PER) return launch_rows<T, W, 256>(ctx, a);
    if constexpr (PER == 8) return launch_rows<T, W, 512>(ctx, a);
    return VA_ERR_UNSUPPORTED;  // (not reached: 256 * 16 is the largest dimension)
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
    VaDeviceGuard on(ctx->device);
    VA_CUDA_TRY(on.err);
    const NormArgs a{x,    residual, weight,   residual_out,    codes, scales,
                     rows, x_stride, residual_stride, dim, group, group ? (dim + group - 1) / group : 1, eps};
    // 16-byte accesses when every row starts on a 16-byte boundary and holds whole vectors.
    const bool wide = dim % 8 == 0 && aligned16(x) && aligned16(weight) && x_stride * es % 16 == 0 &&
                      (!residual || (aligned16(residual) && residual_stride * es % 16 == 0)) &&
                      (!residual_out || aligned16(residual_out)) && ((uintptr_t)codes & 7) == 0;
    if (dtype == VA_DTYPE_BF16)
        return wide ? launch_norm<uint16_t, 16>(ctx, a) : launch_norm<uint16_t, 2>(ctx, a);
    return wide ? launch_norm<float, 16>(ctx, a) : launch_norm<float, 4>(ctx, a);
}

}  // extern "C"
