// Microscaled 4-bit quantisation of a matrix, and back (formats in mx.cuh).
//
// Both are one pass over the data: rows x k elements of 2 or 4 bytes on one side, 17 bytes for 32
// elements on the other: bound by HBM, as long as the instructions an element stay few.  A warp takes
// 512 columns of a row, sixteen a lane (16-byte accesses of the wide side, one 8-byte access of the
// codes), so a block's maximum is one shuffle and the four scale bytes of 128 columns leave as one
// word.  It does so for two rows (four on the way back), all loads before the first use: what depends
// on the columns is worked out once, and the rows' scales lie 16 bytes apart.
#include "mx.cuh"

#include <type_traits>

namespace rfb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// Rows of a warp (51712 x 1536 f16 two 30.7 us, four 31.3, eight 33.7; on the way back 33.3, 32.2, 32.9), and
// columns of a lane and a warp; on the way back eight a lane, so that a warp's 16-byte stores are without gaps.
constexpr int kRows = 2, kLane = 16, kUnit = 32 * kLane;
constexpr int kBackRows = 4, kBackLane = 8, kBackUnit = 32 * kBackLane;

// What a warp works on: R rows (on a boundary of as many) of one of `groups` column groups, group n % groups of
// rows R * (n / groups) on.
struct Units {
    int rows, groups;
    uint64_t magic;  // ceil(2^64 / groups), or 0 for 1: the division is exact for every 32-bit n
    template <int R>
    __device__ __forceinline__ void find(uint32_t n, int& row, int& group) const {
        const uint32_t q = magic ? (uint32_t)__umul64hi(n, magic) : n;
        row = (int)q * R;
        group = (int)(n - q * groups);
    }
};

// Columns [0, COLS) of a row, n of which exist, between memory and a warp's shared memory: a pair at a time where
// the row's address allows, else one.  Neighbouring lanes have neighbouring columns (16384 x 4097 bf16 41 us to codes,
// 37 from them; a lane's own one by one 57 and 190).
template <typename T, int COLS>
struct Ragged {
    using Pair = typename std::conditional<sizeof(T) == 4, uint2, uint32_t>::type;
    using One = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    static __device__ __forceinline__ bool pairs(const T* row) { return ((uintptr_t)row & (2 * sizeof(T) - 1)) == 0; }
    static __device__ __forceinline__ void in(One* buf, const T* row, int n, int lane) {
        const One* r = reinterpret_cast<const One*>(row);
        if (pairs(row)) {
            Pair x[COLS / 64];
#pragma unroll
            for (int j = 0; j < COLS / 64; ++j) {
                const int at = 2 * (j * 32 + lane);
                if (at + 1 < n) x[j] = *reinterpret_cast<const Pair*>(r + at);
                else if constexpr (sizeof(T) == 4) x[j] = make_uint2(at < n ? r[at] : 0u, 0u);
                else x[j] = at < n ? r[at] : 0u;
            }
#pragma unroll
            for (int j = 0; j < COLS / 64; ++j) *reinterpret_cast<Pair*>(buf + 2 * (j * 32 + lane)) = x[j];
        } else {
            One x[COLS / 32];
#pragma unroll
            for (int j = 0; j < COLS / 32; ++j) x[j] = j * 32 + lane < n ? r[j * 32 + lane] : (One)0;
#pragma unroll
            for (int j = 0; j < COLS / 32; ++j) buf[j * 32 + lane] = x[j];
        }
    }
    static __device__ __forceinline__ void out(T* row, const One* buf, int n, int lane) {
        One* r = reinterpret_cast<One*>(row);
        if (pairs(row)) {
#pragma unroll
            for (int j = 0; j < COLS / 64; ++j) {
                const int at = 2 * (j * 32 + lane);
                if (at + 1 < n) *reinterpret_cast<Pair*>(r + at) = *reinterpret_cast<const Pair*>(buf + at);
                else if (at < n) r[at] = buf[at];
            }
        } else {
#pragma unroll
            for (int j = 0; j < COLS / 32; ++j)
                if (j * 32 + lane < n) r[j * 32 + lane] = buf[j * 32 + lane];
        }
    }
};

// The CTAs from `pad_from` on write the zeros of the scales that fill up the last 128 rows.  VEC:
// 16-byte aligned rows and k a multiple of 8.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
k_mx_quantize(const T* src, int ld, int k, uint8_t* codes, int ldc, uint8_t* scales, int kt,
              const Units un, unsigned pad_from) {
    let_next_start();
    wait_previous();
    if (blockIdx.x >= pad_from) {
        mx_pad_scales(scales, un.rows, kt, (blockIdx.x - pad_from) * kThreads + threadIdx.x);
        return;
    }
    __shared__ __align__(16) typename Ragged<T, kUnit>::One buf[VEC ? 1 : kWarps][VEC ? 8 : kRows * kUnit];
    const int lane = threadIdx.x & 31;
    int row, group;
    un.find<kRows>(blockIdx.x * kWarps + (threadIdx.x >> 5), row, group);
    const int rows = un.rows - row;  // of the warp, or more; none behind the last
    if (rows <= 0) return;
    const int col = group * kUnit + lane * kLane;
    const T* p = src + (size_t)row * ld + group * kUnit;
    VecN<T, 8> raw[kRows][2];
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (i < rows && col + 8 * h < k) raw[i][h].load(p + (size_t)i * ld + lane * kLane + 8 * h);
                else raw[i][h].clear();
            }
        }
    } else {
        auto* b = buf[threadIdx.x >> 5];
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            Ragged<T, kUnit>::in(b + i * kUnit, p + (size_t)i * ld, i < rows ? k - group * kUnit : 0, lane);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) raw[i][h].load(reinterpret_cast<const T*>(b + i * kUnit + lane * kLane + 8 * h));
        }
    }
    uint8_t* c = codes + (size_t)row * ldc + (col >> 1);
    uint8_t* s = scales + mx_scale_at(row, (col >> 7) * 4, kt);
    const bool codes_here = col < ((k + 31) & ~31), scale_here = (lane & 7) == 0 && (col >> 7) < kt;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (i >= rows) break;
        float v[2][8];
        raw[i][0].get(v[0]);
        raw[i][1].get(v[1]);
        uint32_t m = max(raw[i][0].amax(), raw[i][1].amax());
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t e = mx_scale_of(m);
        uint32_t word = e << (8 * ((lane >> 1) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        if (codes_here)
            *reinterpret_cast<uint2*>(c + (size_t)i * ldc) = make_uint2(mx_codes8(v[0], e), mx_codes8(v[1], e));
        if (scale_here) *reinterpret_cast<uint32_t*>(s + i * 16) = word;
    }
}

// Eight codes of scale byte e as values of T.
template <typename T>
__device__ __forceinline__ void mx_values8(VecN<T, 8>& x, uint32_t w, uint32_t e) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
    if constexpr (__is_same(T, __half)) {
        // a scale that is a normal f16: the products are rounded once, as from f32
        if (e >= 113 && e <= 142) {
            const uint32_t s = (e - 112) * 0x04000400u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h[j]), *reinterpret_cast<const __half2*>(&s));
                x.w[j] = *reinterpret_cast<const uint32_t*>(&y);
            }
            return;
        }
    }
    const float s = mx_scale_value(e);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&h[j])), make_float2(s, s));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
    x.set(v);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
k_mx_dequantize(const uint8_t* codes, int ldc, const uint8_t* scales, int k, T* dst, int ld,
                int kt, const Units un) {
    __shared__ __align__(16) typename Ragged<T, kBackUnit>::One buf[VEC ? 1 : kWarps][VEC ? 8 : kBackUnit];
    let_next_start();
    wait_previous();
    const int lane = threadIdx.x & 31;
    int row, group;
    un.find<kBackRows>(blockIdx.x * kWarps + (threadIdx.x >> 5), row, group);
    const int rows = un.rows - row;  // of the warp, or more; none behind the last
    if (rows <= 0) return;
    const int first = group * kBackUnit, col = first + lane * kBackLane;
    const uint8_t* c = codes + (size_t)row * ldc + (col >> 1);
    const uint8_t* s = scales + mx_scale_at(row, col >> 5, kt);
    uint32_t w[kBackRows], e[kBackRows];
#pragma unroll
    for (int i = 0; i < kBackRows; ++i) {
        w[i] = 0;
        e[i] = 0;
        if (i < rows && col < k) {
            w[i] = *reinterpret_cast<const uint32_t*>(c + (size_t)i * ldc);
            e[i] = s[i * 16];
        }
    }
    T* to = dst + (size_t)row * ld + first;
#pragma unroll
    for (int i = 0; i < kBackRows; ++i) {
        if (i >= rows) break;
        VecN<T, 8> x;
        if constexpr (!VEC || sizeof(T) == 2) mx_values8(x, w[i], e[i]);
        T* d = to + (size_t)i * ld;
        if constexpr (!VEC) {
            auto* b = buf[threadIdx.x >> 5];
            x.put(reinterpret_cast<T*>(b + lane * kBackLane));
            __syncwarp();
            Ragged<T, kBackUnit>::out(d, b, k - first, lane);
            __syncwarp();
        } else if constexpr (sizeof(T) == 4) {
            // four columns a lane twice, from another's codes, so that the stores are without gaps (4096 x 8192 25.7 us; a
            // lane's own eight 35.9)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = h * 128 + lane * 4, from = h * 16 + (lane >> 1);
                const uint32_t hw = __shfl_sync(0xffffffffu, w[i], from) >> (16 * (lane & 1));
                const float scale = mx_scale_value(__shfl_sync(0xffffffffu, e[i], from));
                const float2 a = e2m1_values(hw & 0xffu), b = e2m1_values((hw >> 8) & 0xffu);
                if (first + at < k)
                    *reinterpret_cast<float4*>(d + at) = make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
            }
        } else {
            if (col < k) x.put(d + lane * kBackLane);
        }
    }
}

bool sizes_ok(int type, int ld, int rows, int k) {
    return mx_type_ok(type) && rows >= 0 && rows <= INT32_MAX - 127 && k >= 1 && k <= INT32_MAX - 511 && ld >= k;
}

// The warps' work in columns of `unit`, and the CTAs it takes; 0 if they are too many.
unsigned make_units(int rows, int k, int rows_each, int unit, Units& u) {
    u.rows = rows;
    u.groups = (k + unit - 1) / unit;
    u.magic = u.groups > 1 ? UINT64_MAX / u.groups + 1 : 0;
    const long long warps = ((long long)rows + rows_each - 1) / rows_each * u.groups;
    return warps <= (long long)UINT32_MAX - kWarps ? (unsigned)((warps + kWarps - 1) / kWarps) : 0;
}

template <typename T>
cudaError_t quantize_t(const void* src, int ld, int rows, int k, uint8_t* codes, int ldc, uint8_t* scales,
                       cudaStream_t st) {
    Units un;
    const unsigned main_ctas = make_units(rows, k, kRows, kUnit, un);
    const int kt = (k + 127) / 128;
    const long long pad_ctas = rows % 128 ? (mx_pad_threads(kt) + kThreads - 1) / kThreads : 0;
    if (main_ctas == 0 || main_ctas + pad_ctas > INT32_MAX) return cudaErrorInvalidValue;
    const bool vec = ptr_aligned(src, 16) && (size_t)ld * sizeof(T) % 16 == 0 && k % 8 == 0;
    auto kern = vec ? k_mx_quantize<T, true> : k_mx_quantize<T, false>;
    return launch_early(mx_start_early(rows, k), kern, dim3((unsigned)(main_ctas + pad_ctas)), kThreads, 0, st, 1, static_cast<const T*>(src), ld, k,
                        codes, ldc, scales, kt, un, main_ctas);
}

template <typename T>
cudaError_t dequantize_t(const uint8_t* codes, int ldc, const uint8_t* scales, int rows, int k, void* dst, int ld,
                         cudaStream_t st) {
    Units un;
    const unsigned ctas = make_units(rows, k, kBackRows, kBackUnit, un);
    if (ctas == 0) return cudaErrorInvalidValue;
    const bool vec = ptr_aligned(dst, 16) && (size_t)ld * sizeof(T) % 16 == 0 && k % 8 == 0;
    auto kern = vec ? k_mx_dequantize<T, true> : k_mx_dequantize<T, false>;
    return launch_early(mx_start_early(rows, k), kern, dim3(ctas), kThreads, 0, st, 1, codes, ldc, scales, k, static_cast<T*>(dst), ld,
                        (k + 127) / 128, un);
}

}  // namespace

cudaError_t mx_quantize(const void* src, int type, int ld, int rows, int k, uint8_t* codes, int ldc, uint8_t* scales,
                        cudaStream_t st) {
    if (!sizes_ok(type, ld, rows, k)) return cudaErrorInvalidValue;
    if (rows == 0) return cudaSuccess;
    if (!src || !ptr_aligned(src, mx_type_size(type)) || !mx_codes_ok(codes, ldc, k) || !scales ||
        !ptr_aligned(scales, 16))
        return cudaErrorInvalidValue;
    switch (type) {
        case MX_F32: return quantize_t<float>(src, ld, rows, k, codes, ldc, scales, st);
        case MX_F16: return quantize_t<__half>(src, ld, rows, k, codes, ldc, scales, st);
        default: return quantize_t<__nv_bfloat16>(src, ld, rows, k, codes, ldc, scales, st);
    }
}

cudaError_t mx_dequantize(const uint8_t* codes, int ldc, const uint8_t* scales, int rows, int k, void* dst, int type,
                          int ld, cudaStream_t st) {
    if (!sizes_ok(type, ld, rows, k)) return cudaErrorInvalidValue;
    if (rows == 0) return cudaSuccess;
    if (!dst || !ptr_aligned(dst, mx_type_size(type)) || !mx_codes_ok(codes, ldc, k) || !scales ||
        !ptr_aligned(scales, 16))
        return cudaErrorInvalidValue;
    switch (type) {
        case MX_F32: return dequantize_t<float>(codes, ldc, scales, rows, k, dst, ld, st);
        case MX_F16: return dequantize_t<__half>(codes, ldc, scales, rows, k, dst, ld, st);
        default: return dequantize_t<__nv_bfloat16>(codes, ldc, scales, rows, k, dst, ld, st);
    }
}

}  // namespace rfb
