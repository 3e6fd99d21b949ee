// va_norm.cu -- root-mean-square norm with the residual's addition and an int8 output with scales.
//
// Per row of `dim` elements (x, residual and weight of one type, fp32 or bf16):
//   h_j    = x_j + residual_j, rounded to the type when it is bf16 (what residual_out stores)
//   z_j    = h_j * weight_j
//   a      = max |z_j| over the row, or over each group of 32, 64 or 128 columns
//   code_j = rint(127 z_j / a)
//   scale  = a / (127 sqrt(mean(h^2) + eps)),   so that code_j * scale ~ z_j / rms(h)
// The rms cancels from the codes, which are therefore exact: the fp32 quotient decides a code
// except within 2^-12 of a border between two codes, where it is redone in fp64 (z has at most 48
// bits), about one element in 2,000. The sum of squares and the scales are fp32. A zero row (or
// group) has codes 0 and scale 0. A row whose sum of squares is not finite, and a group whose a is
// not finite, has codes 0 and scale NaN.
//
// The work is one read of x and residual, one write of residual_out and the codes: HBM-bound. A
// row's elements stay in registers between the statistics and the codes (TPR threads x NV vectors of
// 8 elements), so nothing is read twice; one block barrier per row.
#include <algorithm>

#include "va_internal.cuh"

namespace {

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

// Eight elements starting at p (`n` of them inside the row) as fp32. W is the widest access in bytes
// that every row start allows: 16, or the element's size.
template <typename T, int W>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    if constexpr (W == 16) {
        if constexpr (sizeof(T) == 2) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4*>(p);
            const float4 b = *(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= n) {
                v[i] = 0.f;
            } else if constexpr (sizeof(T) == 2) {
                v[i] = va::bf2f(reinterpret_cast<const uint16_t*>(p)[i]);
            } else {
                v[i] = reinterpret_cast<const float*>(p)[i];
            }
        }
    }
}

template <typename T, int W>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if constexpr (W == 16) {
        if constexpr (sizeof(T) == 2) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = (__float_as_uint(v[2 * i]) >> 16) | (__float_as_uint(v[2 * i + 1]) & 0xFFFF0000u);
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 2)
                    reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(__float_as_uint(v[i]) >> 16);
                else
                    reinterpret_cast<float*>(p)[i] = v[i];
            }
    }
}

// The largest |z| so far, exactly: z = hi + lo with hi = fl(z). Rounding is monotonic, so hi decides
// and lo only breaks ties of hi. Products of two bf16 values fit fp32: lo stays 0.
template <typename T>
struct Top {
    float hi = 0.f, lo = 0.f;
    __device__ __forceinline__ void take(float h, float l) {
        // !(h <= hi): a NaN stays in hi (and is then reported through the scale)
        if constexpr (sizeof(T) == 2) {
            hi = !(h <= hi) ? h : hi;
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

// rint(127 z / a): the fp32 quotient (within 127 * 4 * 2^-24 < 2^-15 of the exact one) unless it is
// within 2^-12 of a border or not finite (127 / a overflowed), then fp64.
template <typename T>
__device__ __forceinline__ int code_of(float h, float w, float inv, const Top<T>& a) {
    const float t = h * w * inv;
    const float r = rintf(t);
    if (fabsf(fabsf(t - r) - 0.5f) >= 0x1p-12f) return (int)r;
    const double z = (double)h * (double)w;
    return (int)rint(z * 127.0 / ((double)a.hi + (double)a.lo));
}

// TPR threads per row, NV vectors of 8 elements per thread; NV * 8 * TPR >= dim. 32-thread rows
// share a block of 128 threads; wider rows take a block each.
template <typename T, int W, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) k_rms_norm_int8(NormArgs a) {
    constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
    constexpr int WARPS = TPR / 32;
    __shared__ float s_sum[ROWS][WARPS], s_hi[ROWS][WARPS], s_lo[ROWS][WARPS];
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const int64_t row_id = (int64_t)blockIdx.x * ROWS + slot;
    const bool live = row_id < a.rows;
    const int64_t row = live ? row_id : a.rows - 1;  // a spare slot repeats the last row, without stores
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const T* weight = static_cast<const T*>(a.weight);

    float h[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = (i * TPR + t) * 8;
        if (j < a.dim) {
            load8<T, W>(x + j, a.dim - j, h[i]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) h[i][k] = 0.f;
        }
    }
    float w[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = (i * TPR + t) * 8;
        if (j < a.dim) {
            load8<T, W>(weight + j, a.dim - j, w[i]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) w[i][k] = 0.f;
        }
    }
    if (res) {
        // Every load precedes the stores: residual_out may be x's or residual's own rows.
        float r[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * TPR + t) * 8;
            if (j < a.dim) load8<T, W>(res + j, a.dim - j, r[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * TPR + t) * 8;
            if (j < a.dim) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    h[i][k] += r[i][k];
                    if constexpr (sizeof(T) == 2) h[i][k] = va::bf2f(va::f2bf_rn(h[i][k]));
                }
                if (live && a.residual_out)
                    store8<T, W>(static_cast<T*>(a.residual_out) + row * a.dim + j, a.dim - j, h[i]);
            }
        }
    }
    float sum = 0.f;
    Top<T> top[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            sum = fmaf(h[i][k], h[i][k], sum);
            top[i].element(h[i][k], w[i][k]);
        }
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
        const int warp = t >> 5;
        if ((t & 31) == 0) {
            s_sum[slot][warp] = sum;
            s_hi[slot][warp] = top[0].hi;
            s_lo[slot][warp] = top[0].lo;
        }
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) sum += s_sum[slot][k];
        if (!a.group) {
#pragma unroll
            for (int k = 0; k < WARPS; ++k) top[0].take(s_hi[slot][k], s_lo[slot][k]);
        }
    }
    if (!live) return;
    const bool finite = sum < INFINITY;  // false for NaN too
    const float per = rsqrtf(sum / (float)a.dim + a.eps) / 127.f;
    int8_t* codes = a.codes + row * a.dim;
    float* scales = a.scales + row * a.groups;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = (i * TPR + t) * 8;
        if (j >= a.dim) continue;
        const Top<T> top_i = a.group ? top[i] : top[0];
        const bool ok = finite && top_i.hi < INFINITY;
        if (a.group ? j % a.group == 0 : j == 0)
            scales[a.group ? j / a.group : 0] = ok ? top_i.hi * per : __int_as_float(0x7FC00000);
        const float inv = 127.f / top_i.hi;
        uint32_t packed[2] = {0u, 0u};
        if (ok && top_i.hi > 0.f) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                packed[k >> 2] |= ((uint32_t)code_of<T>(h[i][k], w[i][k], inv, top_i) & 0xFFu) << (8 * (k & 3));
        }
        if constexpr (W == 16) {
            *reinterpret_cast<uint2*>(codes + j) = make_uint2(packed[0], packed[1]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < a.dim) codes[j + k] = (int8_t)(packed[k >> 2] >> (8 * (k & 3)));
        }
    }
}

template <typename T, int W>
int launch_norm(va_context* ctx, const NormArgs& a) {
    const int vecs = (a.dim + 7) / 8;
    if (vecs <= 64)
        k_rms_norm_int8<T, W, 32, 2><<<(unsigned)((a.rows + 3) / 4), 128, 0, ctx->stream>>>(a);
    else if (vecs <= 256)
        k_rms_norm_int8<T, W, 128, 2><<<(unsigned)a.rows, 128, 0, ctx->stream>>>(a);
    else
        k_rms_norm_int8<T, W, 256, 2><<<(unsigned)a.rows, 256, 0, ctx->stream>>>(a);
    return va_check_launch("k_rms_norm_int8");
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
