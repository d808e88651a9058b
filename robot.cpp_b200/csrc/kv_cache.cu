// kv_cache.cu -- what happens to new tokens before and after attention: rotary positions with several axes, the
// quantised write into the paged cache, and the read back.
//
// All three move bytes: their floor is HBM traffic (rope 2 x rows, write rows + codes, read codes + rows).
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "kv_internal.h"

namespace b2s {

namespace {

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Four consecutive values; the address is aligned to four of them.
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(p) = u;
}

// ------------------------------------------------------------------------------------------------ rotary positions
constexpr int kRopeRows = 4, kRopeThreads = 256, kRopeHalf = 128;

// A block turns kRopeRows rows' heads [h0, h1): the rows' cosines and sines go to shared memory once and serve every
// head, so the double-precision angles cost hd / 2 per row and not per head. The angle is kept in units of pi: its
// reduction is then exact.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRopeThreads)
rope_axes_kernel(const T* x, int64_t ldx, int64_t M, int n_heads, int hd, const int32_t* __restrict__ pos, int64_t ldpos,
                 const __grid_constant__ RopePairs pairs, T* y, int64_t ldy, int heads_per_block) {
    __shared__ float2 cs[kRopeRows][kRopeHalf];
    const int half = hd / 2;
    const int64_t m0 = (int64_t)blockIdx.x * kRopeRows;
    const int rows = (int)min((int64_t)kRopeRows, M - m0);
    griddep_wait();
    griddep_launch();
    for (int e = threadIdx.x; e < rows * half; e += kRopeThreads) {
        const int r = e / half, i = e - r * half;
        double s, c;
        sincospi((double)pos[(m0 + r) * ldpos + pairs.axis[i]] * pairs.turn[i], &s, &c);
        cs[r][i] = make_float2((float)c, (float)s);
    }
    __syncthreads();
    const int h0 = blockIdx.y * heads_per_block, h1 = min(n_heads, h0 + heads_per_block);
    const int step = VEC ? 4 : 1, per_head = half / step, per_row = (h1 - h0) * per_head;
    for (int e = threadIdx.x; e < rows * per_row; e += kRopeThreads) {
        const int r = e / per_row, f = e - r * per_row, h = f / per_head, i = (f - h * per_head) * step;
        const T* xp = x + (m0 + r) * ldx + (int64_t)(h0 + h) * hd + i;
        T* yp = y + (m0 + r) * ldy + (int64_t)(h0 + h) * hd + i;
        if (VEC) {
            const float4 a = load4(xp), b = load4(xp + half);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
            float u[4], w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 t = cs[r][i + j];
                u[j] = __fsub_rn(__fmul_rn(av[j], t.x), __fmul_rn(bv[j], t.y));
                w[j] = __fadd_rn(__fmul_rn(av[j], t.y), __fmul_rn(bv[j], t.x));
            }
            store4(yp, make_float4(u[0], u[1], u[2], u[3]));
            store4(yp + half, make_float4(w[0], w[1], w[2], w[3]));
        } else {
            const float a = (float)xp[0], b = (float)xp[half];
            const float2 t = cs[r][i];
            yp[0] = (T)__fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
            yp[half] = (T)__fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
        }
    }
}

// ------------------------------------------------------------------------------------------------ quantised write
// Code of p = x * (TOP / a).
template <bool E4M3>
__device__ __forceinline__ uint32_t code_of(float p) {
    if (E4M3) return (uint32_t)__nv_cvt_float_to_fp8(p, __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)(int)fminf(fmaxf(roundf(p), -127.0f), 127.0f) & 0xffu;
}

// Lanes of a group share one (token, head, key or value): four values each, so a head of 128 is a warp's 512 bytes.
// Items are ordered (token, key or value, head): consecutive groups read consecutive memory.
template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256)
kv_write_kernel(KvView c, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv, int64_t M,
                const int64_t* __restrict__ slots) {
    const int lane = threadIdx.x % LANES, d = 4 * lane;
    const int64_t groups = (int64_t)gridDim.x * (256 / LANES);
    const int64_t items = M * 2 * c.kv_heads, n_slots = c.n_pages << c.page_shift;
    const bool on = d < c.hd;
    griddep_wait();
    griddep_launch();
    for (int64_t it = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; it < (items + groups - 1) / groups * groups;
         it += groups) {
        const int64_t m = it / (2 * c.kv_heads);
        const int f = (int)(it - m * 2 * c.kv_heads), is_v = f >= c.kv_heads, h = f - is_v * c.kv_heads;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        int64_t slot = -1;
        if (it < items) {
            slot = slots[m];
            if (on) x = load4((is_v ? v + m * ldv : k + m * ldk) + (int64_t)h * c.hd + d);
        }
        float a = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        // an infinity or a NaN anywhere: x - x is NaN for both
        const float z = (x.x - x.x) + (x.y - x.y) + (x.z - x.z) + (x.w - x.w);
        if (z != 0.0f) a = INFINITY;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (slot < 0) continue;
        if (slot >= n_slots) {
            if (lane == 0) atomicOr(&g_device_error, kErrIndex);
            continue;
        }
        const float top = E4M3 ? 448.0f : 127.0f;
        const bool bad = a == INFINITY;
        a = fmaxf(a, 0x1p-100f);
        const float s = bad ? 0.0f : __fdiv_rn(top, a);
        uint32_t w = 0;
        if (!bad)
            w = code_of<E4M3>(__fmul_rn(x.x, s)) | code_of<E4M3>(__fmul_rn(x.y, s)) << 8 |
                code_of<E4M3>(__fmul_rn(x.z, s)) << 16 | code_of<E4M3>(__fmul_rn(x.w, s)) << 24;
        const int64_t row = (((slot >> c.page_shift) * c.kv_heads + h) << c.page_shift) + (slot & ((1 << c.page_shift) - 1));
        if (on) *reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + row * c.hd + d) = w;
        if (lane == 0) (is_v ? c.vs : c.ks)[row] = bad ? __int_as_float(0x7fc00000) : __fdiv_rn(a, top);
    }
}

// ------------------------------------------------------------------------------------------------ read back
template <bool E4M3>
__device__ __forceinline__ float4 values_of(uint32_t w) {
    if (E4M3) {
        const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3));
        const __half2 b = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
        const float2 x = __half22float2(a), y = __half22float2(b);
        return make_float4(x.x, x.y, y.x, y.y);
    }
    return make_float4((float)(int8_t)(w & 0xff), (float)(int8_t)((w >> 8) & 0xff), (float)(int8_t)((w >> 16) & 0xff),
                       (float)(int8_t)(w >> 24));
}

template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256)
kv_read_kernel(KvView c, const int64_t* __restrict__ slots, int64_t M, T* __restrict__ k, int64_t ldk, T* __restrict__ v,
               int64_t ldv) {
    const int lane = threadIdx.x % LANES, d = 4 * lane;
    if (d >= c.hd) return;
    const int parts = (k ? 1 : 0) + (v ? 1 : 0);
    const int64_t groups = (int64_t)gridDim.x * (256 / LANES);
    const int64_t items = M * parts * c.kv_heads, n_slots = c.n_pages << c.page_shift;
    griddep_wait();
    griddep_launch();
    for (int64_t it = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; it < items; it += groups) {
        const int64_t m = it / (parts * c.kv_heads);
        const int f = (int)(it - m * parts * c.kv_heads), second = f >= c.kv_heads, h = f - second * c.kv_heads;
        const bool is_v = !k || second;
        const int64_t slot = slots[m];
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (slot >= n_slots) {
            if (lane == 0) atomicOr(&g_device_error, kErrIndex);
        } else if (slot >= 0) {
            const int64_t row =
                (((slot >> c.page_shift) * c.kv_heads + h) << c.page_shift) + (slot & ((1 << c.page_shift) - 1));
            const float s = (is_v ? c.vs : c.ks)[row];
            x = values_of<E4M3>(*reinterpret_cast<const uint32_t*>((is_v ? c.v : c.k) + row * c.hd + d));
            x = make_float4(__fmul_rn(x.x, s), __fmul_rn(x.y, s), __fmul_rn(x.z, s), __fmul_rn(x.w, s));
        }
        store4((is_v ? v + m * ldv : k + m * ldk) + (int64_t)h * c.hd + d, x);
    }
}

constexpr int64_t kBlocks = 148 * 8;  // 8 blocks of 256 threads fill an SM

template <typename T>
cudaError_t rope_typed(const void* x, int64_t ldx, int64_t M, int n_heads, int hd, const int32_t* pos, int64_t ldpos,
                       const RopePairs& pairs, void* y, int64_t ldy, cudaStream_t st) {
    const int64_t blocks = ceil_div(M, kRopeRows);
    // Few rows: split the heads as well, until the grid has two blocks for each SM.
    int split = (int)ceil_div(2 * 148, blocks);
    if (split > n_heads) split = n_heads;
    const int per = (int)ceil_div(n_heads, split);
    const dim3 grid((unsigned)blocks, (unsigned)ceil_div(n_heads, per));
    const size_t a4 = 4 * sizeof(T) - 1;
    const bool vec = (hd / 2) % 4 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & a4) == 0 &&
                     ldx % 4 == 0 && ldy % 4 == 0;
    if (vec)
        return launch_pdl(rope_axes_kernel<T, true>, grid, dim3(kRopeThreads), st, static_cast<const T*>(x), ldx, M, n_heads,
                          hd, pos, ldpos, pairs, static_cast<T*>(y), ldy, per);
    return launch_pdl(rope_axes_kernel<T, false>, grid, dim3(kRopeThreads), st, static_cast<const T*>(x), ldx, M, n_heads, hd,
                      pos, ldpos, pairs, static_cast<T*>(y), ldy, per);
}

template <typename T, bool E4M3, int LANES>
cudaError_t write_typed(const KvView& c, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t M,
                        const int64_t* slots, cudaStream_t st) {
    const int64_t b = ceil_div(M * 2 * c.kv_heads, 256 / LANES);
    return launch_pdl(kv_write_kernel<T, E4M3, LANES>, dim3((unsigned)(b < kBlocks ? b : kBlocks)), dim3(256), st, c,
                      static_cast<const T*>(k), ldk, static_cast<const T*>(v), ldv, M, slots);
}
template <typename T, bool E4M3, int LANES>
cudaError_t read_typed(const KvView& c, const int64_t* slots, int64_t M, void* k, int64_t ldk, void* v, int64_t ldv,
                       cudaStream_t st) {
    const int64_t b = ceil_div(M * ((k ? 1 : 0) + (v ? 1 : 0)) * c.kv_heads, 256 / LANES);
    return launch_pdl(kv_read_kernel<T, E4M3, LANES>, dim3((unsigned)(b < kBlocks ? b : kBlocks)), dim3(256), st, c, slots, M,
                      static_cast<T*>(k), ldk, static_cast<T*>(v), ldv);
}

// Lanes for a head of hd values, four each: a power of two that divides a warp.
#define KV_LANES(fn, T, E, ...)                              \
    (c.hd > 64   ? fn<T, E, 32>(__VA_ARGS__)                 \
     : c.hd > 32 ? fn<T, E, 16>(__VA_ARGS__)                 \
                 : fn<T, E, 8>(__VA_ARGS__))
#define KV_TYPES(fn, ...)                                                                                        \
    (bf16 ? (c.e4m3 ? KV_LANES(fn, __nv_bfloat16, true, __VA_ARGS__) : KV_LANES(fn, __nv_bfloat16, false, __VA_ARGS__)) \
          : (c.e4m3 ? KV_LANES(fn, float, true, __VA_ARGS__) : KV_LANES(fn, float, false, __VA_ARGS__)))

}  // namespace

cudaError_t launch_rope_axes(bool bf16, const void* x, int64_t ldx, int64_t M, int n_heads, int hd, const int32_t* pos,
                             int64_t ldpos, const RopePairs& pairs, void* y, int64_t ldy, cudaStream_t st) {
    if (M <= 0) return cudaSuccess;
    return bf16 ? rope_typed<__nv_bfloat16>(x, ldx, M, n_heads, hd, pos, ldpos, pairs, y, ldy, st)
                : rope_typed<float>(x, ldx, M, n_heads, hd, pos, ldpos, pairs, y, ldy, st);
}

cudaError_t launch_kv_write(const KvView& c, bool bf16, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t M,
                            const int64_t* slots, cudaStream_t st) {
    if (M <= 0) return cudaSuccess;
    return KV_TYPES(write_typed, c, k, ldk, v, ldv, M, slots, st);
}

cudaError_t launch_kv_read(const KvView& c, const int64_t* slots, int64_t M, bool bf16, void* k, int64_t ldk, void* v,
                           int64_t ldv, cudaStream_t st) {
    if (M <= 0 || (!k && !v)) return cudaSuccess;
    return KV_TYPES(read_typed, c, slots, M, k, ldk, v, ldv, st);
}

}  // namespace b2s
