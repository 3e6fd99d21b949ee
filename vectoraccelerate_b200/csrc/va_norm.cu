// va_norm.cu -- root-mean-square norm with the residual's addition and an int8 output with scales.
//
// Per row of `dim` elements (x, residual and weight of one type, fp32 or bf16):
//   h_j    = x_j + residual_j, rounded to the type when it is bf16 (what residual_out stores)
//   z_j    = h_j * weight_j
//   a      = max |z_j| over the row, or over each group of 32, 64 or 128 columns
//   code_j = rint(127 z_j / a)
//   scale  = a / (127 sqrt(mean(h^2) + eps)),   so that code_j * scale ~ z_j / rms(h)
// The rms cancels from the codes, which are therefore exact: the fp32 quotient decides a code
// except within 2^-12 of a border between two codes (one element in 2,000), where the exact
// remainder does. The sum of squares and the scales are fp32. A row (or group) with
// a < 2^-80 has codes 0 and scale 0. A row whose sum of squares is not finite, and a group whose a is
// not finite, has codes 0 and scale NaN.
//
// The work is one read of x and residual, one write of residual_out and the codes: HBM-bound, with
// ~20 instructions per element to hide. A thread holds 8 neighbouring elements of a row in registers between
// the statistics and the codes, so nothing is read twice. Blocks are persistent: each thread's vectors of
// the next rows come through cp.async into shared memory of its own (no barrier), the weights stay in
// registers, and a row costs one block barrier.
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

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// The largest |z| so far, exactly: z = hi + lo with hi = fl(z). Rounding is monotonic, so hi decides
// and lo only breaks ties of hi. Products of two bf16 values fit fp32: lo stays 0. A NaN stays in hi (and
// is then reported through the scale).
template <typename T>
struct Top {
    float hi = 0.f, lo = 0.f;
    __device__ __forceinline__ void take(float h, float l) {
        if constexpr (sizeof(T) == 2) {
            hi = max_nan(hi, h);
        } else {
            const bool more = !(h <= hi) || (h == hi && l > lo);
            lo = more ? l : lo;
            hi = more ? h : hi;
        }
    }
    __device__ __forceinline__ void element(float h, float w) {
        const float z = h * w;
        if constexpr (sizeof(T) == 2) {
            take(fabsf(z), 0.f);
        } else {
            const float e = fmaf(h, w, -z);
            take(fabsf(z), z < 0.f ? -e : e);
        }
    }
    template <int WIDTH>
    __device__ __forceinline__ void lanes() {
#pragma unroll
        for (int o = 1; o < WIDTH; o <<= 1) {
            const float h = __shfl_xor_sync(0xFFFFFFFFu, hi, o);
            const float l = sizeof(T) == 2 ? 0.f : __shfl_xor_sync(0xFFFFFFFFu, lo, o);
            take(h, l);
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

// rint(127 z / a) of eight elements, packed. t = z (127 / a) in fp32 is within 127 * 4 * 2^-24 < 2^-15 of the
// quotient; adding 1.5 * 2^23 rounds it (to even) into the low byte. Where some t is within 2^-12 of the border
// b between two codes, the sign of 127 z - b a decides: for bf16 both products are exact in fp32 (7 + 16 and 8 + 16
// bits); for fp32 their rounding errors and the low parts are added (48 bits).
template <typename T>
__device__ __forceinline__ uint2 codes_of(const Vec<T>& h, const Vec<T>& w, const Top<T>& a) {
    uint32_t m[8];
    constexpr float SHIFT = 12582912.f;
    const float inv = 127.f / a.hi;
    float off = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float t = h[k] * w[k] * inv, r = t + SHIFT;
        m[k] = __float_as_uint(r);
        off = fmaxf(off, fabsf(t - (r - SHIFT)));
    }
    if (off > 0.5f - 0x1p-12f) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float z = h[k] * w[k], t = z * inv, r = __uint_as_float(m[k]) - SHIFT, d = t - r;
            if (fabsf(d) > 0.5f - 0x1p-12f) {
                const float b = r + copysignf(0.5f, d), p = b * a.hi, q = 127.f * z;
                float diff = q - p;
                if constexpr (sizeof(T) == 4)
                    diff += (fmaf(127.f, z, -q) - fmaf(b, a.hi, -p)) + (127.f * fmaf(h[k], w[k], -z) - b * a.lo);
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

// Rows on their way per thread (16-byte accesses only).
template <typename T>
constexpr int stages_of() { return sizeof(T) == 2 ? 3 : 2; }

// TPR threads per row, 8 elements each; 8 * TPR >= dim. Narrow rows share a block of 128 threads.
template <typename T, int W, int TPR>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR < 512 ? 1024 / (TPR < 128 ? 128 : TPR) : 2)
    k_rms_norm_int8(NormArgs a) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, ROWS = THREADS / TPR, WARPS = TPR / 32, STAGES = stages_of<T>();
    constexpr int HALVES = sizeof(T) / 2;  // 16-byte pieces of a vector
    extern __shared__ uint4 s_in[];        // [stage][x, residual][piece][thread]
    __shared__ float s_sum[2][ROWS][WARPS], s_hi[2][ROWS][WARPS], s_lo[2][ROWS][WARPS];
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, j = t * 8;
    const Vec<T> w = load8<T, W>(static_cast<const T*>(a.weight) + j, a.dim - j);
    const int64_t step = (int64_t)gridDim.x * ROWS;
    // Every thread of a block makes the same number of turns (barriers); rows past the end repeat the last one.
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    const auto mine = [&](int64_t r) { return min(r + slot, a.rows - 1); };
    const auto fetch = [&](int64_t r, int stage) {
        if constexpr (W == 16) {
            if (r < a.rows && j < a.dim) {
                const T* px = static_cast<const T*>(a.x) + mine(r) * a.x_stride + j;
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(s_in + (size_t)stage * 2 * HALVES * THREADS + threadIdx.x);
#pragma unroll
                for (int i = 0; i < HALVES; ++i) cp_async16(dst + i * THREADS * 16, reinterpret_cast<const uint4*>(px) + i);
                if (a.residual) {
                    const T* pr = static_cast<const T*>(a.residual) + mine(r) * a.residual_stride + j;
#pragma unroll
                    for (int i = 0; i < HALVES; ++i)
                        cp_async16(dst + (HALVES + i) * THREADS * 16, reinterpret_cast<const uint4*>(pr) + i);
                }
            }
            cp_async_commit();
        }
    };
    const auto take = [&](int64_t r, int stage, bool residual) {
        if constexpr (W == 16) {
            Vec<T> v;
            const uint4* from = s_in + ((size_t)stage * 2 + (residual ? 1 : 0)) * HALVES * THREADS + threadIdx.x;
#pragma unroll
            for (int i = 0; i < HALVES; ++i) {
                const uint4 u = j < a.dim ? from[i * THREADS] : make_uint4(0u, 0u, 0u, 0u);
                v.w[4 * i] = u.x, v.w[4 * i + 1] = u.y, v.w[4 * i + 2] = u.z, v.w[4 * i + 3] = u.w;
            }
            return v;
        } else {
            const T* p = residual ? static_cast<const T*>(a.residual) + mine(r) * a.residual_stride
                                  : static_cast<const T*>(a.x) + mine(r) * a.x_stride;
            return load8<T, W>(p + j, a.dim - j);
        }
    };
    for (int s = 0; s < STAGES - 1; ++s) fetch(row0 + s * step, s);
    int stage = 0, turn = 0;
    for (int64_t r = row0; r < a.rows; r += step, turn ^= 1) {
        // (residual_out may be x's or residual's own rows: a row is stored only after its loads.)
        fetch(r + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
        cp_async_wait<STAGES - 1>();
        const int64_t row = mine(r);
        const bool live = r + slot < a.rows;
        Vec<T> h = take(r, stage, false);
        if (a.residual) {
            const Vec<T> v = take(r, stage, true);
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int k = 0; k < 4; ++k) h.w[k] = pack_bf16(h[2 * k] + v[2 * k], h[2 * k + 1] + v[2 * k + 1]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) h.w[k] = __float_as_uint(h[k] + v[k]);
            }
            if (a.residual_out && live && j < a.dim)
                store8<T, W>(static_cast<T*>(a.residual_out) + row * a.dim + j, a.dim - j, h);
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        float sum = 0.f;
        Top<T> top;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            sum = fmaf(h[k], h[k], sum);
            top.element(h[k], w[k]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (a.group)
            top.lanes(a.group / 8);
        else
            top.template lanes<32>();
        if constexpr (WARPS > 1) {
            // Two sets of slots in turn: one barrier per row.
            if ((t & 31) == 0) {
                s_sum[turn][slot][t >> 5] = sum;
                s_hi[turn][slot][t >> 5] = top.hi;
                s_lo[turn][slot][t >> 5] = top.lo;
            }
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) sum += s_sum[turn][slot][k];
            if (!a.group) {
#pragma unroll
                for (int k = 0; k < WARPS; ++k) top.take(s_hi[turn][slot][k], s_lo[turn][slot][k]);
            }
        }
        if (!live || j >= a.dim) continue;
        const bool ok = sum < INFINITY && top.hi < INFINITY;  // false for NaN too
        if (a.group ? j % a.group == 0 : j == 0) {
            const float per = rsqrtf(sum / (float)a.dim + a.eps) / 127.f;
            a.scales[row * a.groups + (a.group ? j / a.group : 0)] =
                !ok ? __int_as_float(0x7FC00000) : top.hi >= SMALLEST ? top.hi * per : 0.f;
        }
        uint2 packed = make_uint2(0u, 0u);
        if (ok && top.hi >= SMALLEST) packed = codes_of<T>(h, w, top);
        int8_t* codes = a.codes + row * a.dim + j;
        if constexpr (W == 16) {
            *reinterpret_cast<uint2*>(codes) = packed;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < a.dim) codes[k] = (int8_t)((k < 4 ? packed.x : packed.y) >> (8 * (k & 3)));
        }
    }
}

template <typename T, int W, int TPR>
int launch_rows(va_context* ctx, const NormArgs& a) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, ROWS = THREADS / TPR, BLOCKS = TPR < 512 ? 1024 / THREADS : 2;
    constexpr size_t SMEM = W == 16 ? (size_t)stages_of<T>() * 2 * (sizeof(T) / 2) * THREADS * 16 : 0;
    if (SMEM > 47 * 1024)  // (with the static part over the 48 KB that need no asking)
        VA_CUDA_TRY(cudaFuncSetAttribute(k_rms_norm_int8<T, W, TPR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    const int64_t grid = std::min<int64_t>((a.rows + ROWS - 1) / ROWS, (int64_t)ctx->sm_count * BLOCKS);
    k_rms_norm_int8<T, W, TPR><<<(unsigned)grid, THREADS, SMEM, ctx->stream>>>(a);
    return va_check_launch("k_rms_norm_int8");
}

template <typename T, int W>
int launch_norm(va_context* ctx, const NormArgs& a) {
    if (a.dim <= 256) return launch_rows<T, W, 32>(ctx, a);
    if (a.dim <= 512) return launch_rows<T, W, 64>(ctx, a);
    if (a.dim <= 1024) return launch_rows<T, W, 128>(ctx, a);
    if (a.dim <= 2048) return launch_rows<T, W, 256>(ctx, a);
    return launch_rows<T, W, 512>(ctx, a);
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
