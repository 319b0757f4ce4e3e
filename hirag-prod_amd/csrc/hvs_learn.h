// Device and host helpers shared by the learning kernels (hvs_adapters.hip, hvs_feedback.hip): element access for the
// three dtypes, 16-byte chunks with guards, wave sums, the current-device guard.
#pragma once
#include <atomic>
#include <mutex>

#include "hvs_gemm_tile.h"

template <int DT> struct Elem;
template <> struct Elem<HVS_F32> {
    typedef float type;
    typedef f32x4 loose __attribute__((aligned(4)));  // 16 bytes at an element's address
    static constexpr int EPC = 4;  // elements per 16-byte chunk
};
template <> struct Elem<HVS_F16> {
    typedef _Float16 type;
    typedef f32x4 loose __attribute__((aligned(2)));
    static constexpr int EPC = 8;
};
template <> struct Elem<HVS_BF16> {
    typedef __bf16 type;
    typedef f32x4 loose __attribute__((aligned(2)));
    static constexpr int EPC = 8;
};

__device__ __forceinline__ float learn_to_float(float v) { return v; }
__device__ __forceinline__ float learn_to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float learn_to_float(__bf16 v) { return hvs_bf16_to_float(__builtin_bit_cast(uint16_t, v)); }
template <typename E> __device__ __forceinline__ E learn_from_float(float v);
template <> __device__ __forceinline__ float learn_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 learn_from_float<_Float16>(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ __bf16 learn_from_float<__bf16>(float v) { return __builtin_bit_cast(__bf16, hvs_float_to_bf16(v)); }

// elements k .. k + EPC - 1 of a row of K elements, zeros past its end.  ALIGNED: the row starts on 16 bytes, K and k are
// multiples of EPC; otherwise the same 16-byte load from an address that is a multiple of the element's size only (global
// memory takes those), and the row's end element by element.
template <int DT, bool ALIGNED> __device__ __forceinline__ f32x4 load_chunk(const void *row, int k, int K) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC;
    typedef typename Elem<DT>::loose loose;
    const E *p = reinterpret_cast<const E *>(row);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (ALIGNED) {
        if (k < K) v = *reinterpret_cast<const f32x4 *>(p + k);
    } else if (k + EPC <= K) {
        v = *reinterpret_cast<const loose *>(p + k);
    } else if (k < K) {
        E e[EPC];
#pragma unroll
        for (int i = 0; i < EPC; i++) e[i] = k + i < K ? p[k + i] : (E)0.0f;
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

template <int DT> __device__ __forceinline__ void chunk_to_float(const f32x4 &c, float *out) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC;
    typedef E vec __attribute__((ext_vector_type(EPC)));
    const vec v = __builtin_bit_cast(vec, c);
#pragma unroll
    for (int i = 0; i < EPC; i++) out[i] = learn_to_float((E)v[i]);
}

// D(16 x 16) += A(16 x 4 EPC) B(16 x 4 EPC)^T: lane (m = lane & 15, g = lane >> 4) holds the chunk k = EPC g .. of row m of
// both operands; D: row 4 g + reg (an A row), column lane & 15 (a B row).  fp32: four 16x16x4 steps pair element j of the chunks.
template <int DT> __device__ __forceinline__ f32x4 mfma_chunk(const f32x4 &a, const f32x4 &b, f32x4 c) {
    if (DT == HVS_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    if (DT == HVS_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// A 16-row, 64-byte piece of a row matrix on its way to mfma_chunk.  Lane l LOADS chunk l & 3 of row l >> 2 (four lanes cover 64
// bytes of a row: the vector memory path takes such a quad in one cycle; fragment order, 16 rows next to each other, costs
// it four) and the lanes trade their chunks through 1 KB of LDS of their wave's own.  No barrier: a wave's LDS accesses stay in order.
__device__ __forceinline__ int turn_row(int lane) { return lane >> 2; }
template <int DT> __device__ __forceinline__ int turn_k(int lane) { return (lane & 3) * Elem<DT>::EPC; }
__device__ __forceinline__ void turn_put(char *lds, const f32x4 &v, int lane) {
    const int r = lane >> 2;
    *reinterpret_cast<f32x4 *>(lds + (r * 4 + ((lane & 3) ^ (r >> 2))) * 16) = v;
}
__device__ __forceinline__ f32x4 turn_get(const char *lds, int lane) {
    const int m = lane & 15;
    return *reinterpret_cast<const f32x4 *>(lds + (m * 4 + ((lane >> 4) ^ (m >> 2))) * 16);
}

__device__ __forceinline__ float learn_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <int CTRL> __device__ __forceinline__ float learn_dpp(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// Two sums (or two largest values) over the wave at once, in vector registers alone: the halves trade places, so that each works on
// one value; rows of 16 lanes are joined by rotation, then the two rows of a half.  a and b become the results, the same in every lane.
struct LearnAdd {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct LearnMax {  // of a number and a NaN: the number
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
template <class OP> __device__ __forceinline__ void learn_wave_join2(float &a, float &b, OP op) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    float u = op(__uint_as_float(r[0]), __uint_as_float(r[1]));  // lanes 0-31: a, lanes 32-63: b
    u = op(u, learn_dpp<0x128>(u));                              // rotations by 8, 4, 2, 1
    u = op(u, learn_dpp<0x124>(u));
    u = op(u, learn_dpp<0x122>(u));
    u = op(u, learn_dpp<0x121>(u));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(u), __float_as_uint(u), false, false);
    const uint32_t s = __float_as_uint(op(__uint_as_float(r[0]), __uint_as_float(r[1])));
    a = __uint_as_float(__builtin_amdgcn_readlane(s, 0));
    b = __uint_as_float(__builtin_amdgcn_readlane(s, 32));
}
__device__ __forceinline__ void learn_wave_sum2(float &a, float &b) { learn_wave_join2(a, b, LearnAdd()); }
__device__ __forceinline__ void learn_wave_max2(float &a, float &b) { learn_wave_join2(a, b, LearnMax()); }

// Makes `device` current for a call and the caller's device current again after it.
struct DeviceGuard {
    int before = -1;
    hipError_t status;
    explicit DeviceGuard(int device) {
        status = hipGetDevice(&before);
        if (status == hipSuccess && device != before) status = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// Lets a kernel have `lds` bytes of dynamic LDS on the current device.  Below 48 KB nothing is asked; the request (a microsecond)
// is made again only where the kernel has not been allowed as much on that device yet.
template <auto *KERNEL> static int learn_allow_lds(int lds) {
    static std::atomic<int> allowed[16];
    static std::mutex asking;  // a request for less must not follow one for more
    if (lds <= 48 * 1024) return 0;
    int device = 0;
    HVS_HIP(hipGetDevice(&device));
    HVS_REQUIRE(device < 16, "device %d: at most 16 are served", device);
    if (allowed[device].load(std::memory_order_acquire) >= lds) return 0;
    const std::lock_guard<std::mutex> lock(asking);
    if (allowed[device].load(std::memory_order_acquire) >= lds) return 0;
    HVS_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    allowed[device].store(lds, std::memory_order_release);
    return 0;
}

static inline bool learn_dtype_ok(int dt) { return dt == HVS_F32 || dt == HVS_F16 || dt == HVS_BF16; }
static inline bool learn_aligned(const void *p, int64_t ld_bytes, int64_t row_bytes) {
    return ((uintptr_t)p & 15) == 0 && (ld_bytes & 15) == 0 && (row_bytes & 15) == 0;
}
// rows_a rows of row_a bytes at pitch ld_a and the same of b share a byte.  Columns of one wide tensor do not; rows of different
// pitches count as sharing where the ranges they span do.
static inline bool learn_overlap(const void *a, int64_t rows_a, int64_t ld_a, int64_t row_a, const void *b, int64_t rows_b, int64_t ld_b, int64_t row_b) {
    if (rows_a <= 0 || rows_b <= 0) return false;
    const uintptr_t a0 = (uintptr_t)a, a1 = a0 + (uintptr_t)((rows_a - 1) * ld_a + row_a);
    const uintptr_t b0 = (uintptr_t)b, b1 = b0 + (uintptr_t)((rows_b - 1) * ld_b + row_b);
    if (a0 >= b1 || b0 >= a1) return false;
    if (ld_a != ld_b || ld_a <= 0) return true;
    const int64_t ahead = (int64_t)(b0 - a0) % ld_a, d = ahead < 0 ? ahead + ld_a : ahead;  // from a row of a to the next row of b
    return d < row_a || d + row_b > ld_a;
}
// sizes of a workspace carved in 256-byte steps
struct WorkspaceCut {
    char *base;
    uint64_t used = 0;
    explicit WorkspaceCut(void *p) : base((char *)p) {}
    template <typename P> P *take(uint64_t bytes) {
        P *p = reinterpret_cast<P *>(base + used);
        used += (bytes + 255) & ~(uint64_t)255;
        return p;
    }
};
