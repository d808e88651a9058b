// kv_cache.cu -- what happens to new tokens before and after attention: rotary positions with several axes, the
// quantised write into the paged cache, and the read back.
//
// All three move bytes: their floor is HBM traffic (rope 2 x rows, write rows + codes, read codes + rows). Measured (the copy
// rate is 6.5 TB/s): rope, 16384 bf16 rows of 25 heads of 128, 37.8 us, 5.6 TB/s; write, 18432 bf16 tokens of 5 + 5 heads to
// e4m3, 16.8 us, 4.2 TB/s; read, 65537 tokens of 8 + 8 e4m3 heads to bf16, 76 us, 5.3 TB/s; a few rows 2-3 us, one launch.
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

// Eight consecutive values; the address is aligned to 16 bytes.
struct F8 {
    float v[8];
};
// Eight elements as they lie in memory, their values, and the largest magnitude's bits (0x7f800000 or more: an infinity or NaN).
template <typename T>
struct Raw8 {
    uint4 u[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
__device__ __forceinline__ F8 values(const Raw8<float>& r) {
    return F8{{__uint_as_float(r.u[0].x), __uint_as_float(r.u[0].y), __uint_as_float(r.u[0].z), __uint_as_float(r.u[0].w),
               __uint_as_float(r.u[1].x), __uint_as_float(r.u[1].y), __uint_as_float(r.u[1].z), __uint_as_float(r.u[1].w)}};
}
__device__ __forceinline__ F8 values(const Raw8<__nv_bfloat16>& x) {
    const uint32_t w[4] = {x.u[0].x, x.u[0].y, x.u[0].z, x.u[0].w};
    F8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.v[2 * i] = __uint_as_float(w[i] << 16);
        r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return r;
}
__device__ __forceinline__ uint32_t magnitude(const Raw8<float>& r) {
    uint32_t b = 0;
    const F8 x = values(r);
#pragma unroll
    for (int j = 0; j < 8; ++j) b = max(b, __float_as_uint(x.v[j]) & 0x7fffffffu);
    return b;
}
__device__ __forceinline__ uint32_t magnitude(const Raw8<__nv_bfloat16>& r) {
    const uint32_t m = 0x7fff7fffu;
    const uint32_t b = __vmaxu2(__vmaxu2(r.u[0].x & m, r.u[0].y & m), __vmaxu2(r.u[0].z & m, r.u[0].w & m));
    return max(b << 16, b & 0xffff0000u);
}
__device__ __forceinline__ void store8(float* p, const F8& x) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const F8& x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x.v[2 * i], x.v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------------------------------------ rotary positions
__device__ __forceinline__ uint4 pack16(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack16(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void unpack16(uint4 u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack16(uint4 u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Cosine and sine of pos * turn (units of pi). The product and its reduction to [-1, 1] are double, the reduction is exact;
// the remainder goes on as a float and its rest r, with sin(h + r) = sin h + r cos h. Each is within 1.5 * 2^-24 (the float
// functions' one unit in the last place, then one rounding). In double throughout the functions took as long as the rows.
__device__ __forceinline__ float2 cos_sin(int pos, double turn) {
    const double t = (double)pos * turn, r = t - 2.0 * rint(0.5 * t);
    const float h = (float)r, l = (float)(r - (double)h) * 3.14159265f;
    float s, c;
    sincospif(h, &s, &c);
    return make_float2(__fmaf_rn(-l, s, c), __fmaf_rn(l, c, s));
}

// A warp turns one row's heads [h0, h0 + heads): per_head lanes of W pairs (16 bytes and the 16 half a head on) hold their
// cosines and sines in registers for all of them, 32 / per_head heads side by side, kRopeFlight of those steps in flight; the
// angles are formed while the first ones arrive. One thread a pair of values had taken 50.8 us for the
// 16384 rows.
constexpr int kRopeFlight = 4;
template <typename T, int W>
__global__ void __launch_bounds__(256)
rope_axes_kernel(const T* x, int64_t ldx, int M, int n_heads, int hd, const int32_t* __restrict__ pos, int64_t ldpos,
                 const __grid_constant__ RopePairs pairs, T* y, int64_t ldy, int heads_per_warp, int warps_a_row) {
    const int half = hd / 2, per_head = half / W, G = 32 / per_head;
    const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), row = w / (uint32_t)warps_a_row;
    const int lane = threadIdx.x & 31, g = lane / per_head, i = (lane - g * per_head) * W;
    const int h0 = (int)(w - row * (uint32_t)warps_a_row) * heads_per_warp, h1 = min(n_heads, h0 + heads_per_warp);
    griddep_wait();
    griddep_launch();
    if (row >= (uint32_t)M || g >= G) return;
    const T* xr = x + row * ldx + i;
    T* yr = y + row * ldy + i;
    float2 cs[W];
    bool angles = false;
    for (int h = h0 + g; h < h1; h += G * kRopeFlight) {
        uint4 a[kRopeFlight], b[kRopeFlight];
#pragma unroll
        for (int k = 0; k < kRopeFlight; ++k) {
            const int64_t at = (int64_t)min(h + k * G, h1 - 1) * hd;  // past the end the last head once more, not written
            a[k] = *reinterpret_cast<const uint4*>(xr + at);
            b[k] = *reinterpret_cast<const uint4*>(xr + at + half);
        }
        if (!angles) {
            angles = true;
#pragma unroll
            for (int j = 0; j < W; ++j) cs[j] = cos_sin(pos[row * ldpos + pairs.axis[i + j]], pairs.turn[i + j]);
        }
#pragma unroll
        for (int k = 0; k < kRopeFlight; ++k) {
            if (h + k * G >= h1) break;
            float u[W], v[W], p[W], q[W];
            unpack16(a[k], u);
            unpack16(b[k], v);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                p[j] = __fsub_rn(__fmul_rn(u[j], cs[j].x), __fmul_rn(v[j], cs[j].y));
                q[j] = __fadd_rn(__fmul_rn(u[j], cs[j].y), __fmul_rn(v[j], cs[j].x));
            }
            const int64_t at = (int64_t)(h + k * G) * hd;
            *reinterpret_cast<uint4*>(yr + at) = pack16(p);
            *reinterpret_cast<uint4*>(yr + at + half) = pack16(q);
        }
    }
}

// Any alignment and any half: one pair a thread and step, cosines and sines of a block's rows in shared memory.
constexpr int kRopeRows = 4, kRopeHalf = 128;
template <typename T>
__global__ void __launch_bounds__(256)
rope_axes_any_kernel(const T* x, int64_t ldx, int64_t M, int n_heads, int hd, const int32_t* __restrict__ pos, int64_t ldpos,
                     const __grid_constant__ RopePairs pairs, T* y, int64_t ldy) {
    __shared__ float2 cs[kRopeRows][kRopeHalf];
    const int half = hd / 2;
    const int64_t m0 = (int64_t)blockIdx.x * kRopeRows;
    const int rows = (int)min((int64_t)kRopeRows, M - m0);
    griddep_wait();
    griddep_launch();
    for (int e = threadIdx.x; e < rows * half; e += 256) {
        const int r = e / half, i = e - r * half;
        cs[r][i] = cos_sin(pos[(m0 + r) * ldpos + pairs.axis[i]], pairs.turn[i]);
    }
    __syncthreads();
    const int per_row = n_heads * half;
    for (int r = 0; r < rows; ++r) {
        for (int e = threadIdx.x; e < per_row; e += 256) {
            const int h = e / half, i = e - h * half;
            const T* p = x + (m0 + r) * ldx + (int64_t)h * hd + i;
            T* q = y + (m0 + r) * ldy + (int64_t)h * hd + i;
            const float a = (float)p[0], b = (float)p[half];
            const float2 t = cs[r][i];
            q[0] = (T)__fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
            q[half] = (T)__fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
        }
    }
}

// ------------------------------------------------------------------------------------------------ quantised write
// Codes of eight x * s, packed.
template <bool E4M3>
__device__ __forceinline__ uint2 codes_of(const F8& x, float s) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __fmul_rn(x.v[4 * i + j], s);
        if (E4M3) {
            w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(p[0], p[1]), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(p[2], p[3]), __NV_SATFINITE, __NV_E4M3) << 16;
        } else {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)  // |p| + 1/2 rounded towards zero has the whole part of the exact sum; |p| < 127.5
                w[i] |= ((uint32_t)(int)__fadd_rz(p[j], copysignf(0.5f, p[j])) & 0xffu) << (8 * j);
        }
    }
    return make_uint2(w[0], w[1]);
}

// LANES (4, 8 or 16) lanes share one row (a head of a key or a value), eight values each. A warp takes one head a step for each of
// its 32 / LANES groups, from one token's 2 kv_heads: the loads of all its steps are in flight before the first is used, and the
// lanes of a group hold one step's scale each. 18432 bf16 tokens of 5 + 5 heads of 128 to e4m3 (the bytes alone: 10.9 us): 23.9
// us with one step, 20.9 with two, 21.1 with four (of which the fourth is empty), 16.8 with five (4.2 TB/s), 17.0 with six; of
// 8 + 8 heads 41, 33, 29.6, 29.8 and 30 us. What is left is issue slots and latency: 56 registers hold 32 warps an SM, and
// 40 registers, which hold 48, took 17.8 us.
template <int LANES>
constexpr int kWriteSteps = LANES < 5 ? LANES : 5;
template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256)
kv_write_kernel(KvView c, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv, int M,
                const int64_t* __restrict__ slots, int warps_a_token) {
    constexpr int G = 32 / LANES;
    const int lane = threadIdx.x % LANES, g = (threadIdx.x & 31) / LANES, d = 8 * lane;
    const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), token = w / (uint32_t)warps_a_token;
    const int64_t m = token;
    // heads f0, f0 + step, ...: a token's warps have the same number of them
    const int f0 = (int)(w - token * (uint32_t)warps_a_token) * G + g, step = warps_a_token * G, heads = 2 * c.kv_heads;
    griddep_wait();
    griddep_launch();
    if (m >= M) return;
    const int64_t slot = slots[m];  // looked at when the rows are on their way
    const int end = heads - (f0 - g);  // the warp's steps end there
    Raw8<T> x[kWriteSteps<LANES>];
#pragma unroll
    for (int i = 0; i < kWriteSteps<LANES>; ++i) {
        const int f = f0 + i * step;
        x[i] = Raw8<T>{};
        if (f < heads && d < c.hd)
            x[i] = load8(f < c.kv_heads ? k + m * ldk + (int64_t)f * c.hd + d : v + m * ldv + (int64_t)(f - c.kv_heads) * c.hd + d);
    }
    if (slot < 0) return;
    if (slot >= c.n_pages << c.page_shift) {
        if (f0 == 0 && lane == 0) atomicOr(&g_device_error, kErrIndex);
        return;
    }
    const int64_t row0 = (((slot >> c.page_shift) * c.kv_heads) << c.page_shift) + (slot & ((1 << c.page_shift) - 1));
    auto row_of = [&](int f) { return row0 + ((int64_t)(f < c.kv_heads ? f : f - c.kv_heads) << c.page_shift); };
    // the scales of the warp's heads: lane i of a group has step i's
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kWriteSteps<LANES>; ++i) {
        if (i * step >= end) break;
        uint32_t bits = magnitude(x[i]);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
        if (lane == i) mine = bits;
    }
    constexpr float top = E4M3 ? 448.0f : 127.0f, by_top = 1.0f / top;
    const bool bad = mine >= 0x7f800000u;
    const float a = bad ? 1.0f : fmaxf(__uint_as_float(mine), 0x1p-100f);
    const float up = bad ? 0.0f : __fdiv_rn(top, a);
    if (lane < kWriteSteps<LANES> && f0 + lane * step < heads) {
        // a / top, correctly rounded: the quotient by the rounded reciprocal, corrected once by its exact remainder (Markstein's theorem)
        const float q0 = __fmul_rn(a, by_top), quotient = __fmaf_rn(__fmaf_rn(-q0, top, a), by_top, q0);
        const int f = f0 + lane * step;
        (f < c.kv_heads ? c.ks : c.vs)[row_of(f)] = bad ? __int_as_float(0x7fc00000) : quotient;
    }
#pragma unroll
    for (int i = 0; i < kWriteSteps<LANES>; ++i) {
        if (i * step >= end) break;
        const int f = f0 + i * step;
        const float by = __shfl_sync(0xffffffffu, up, i, LANES);
        if (f >= heads || d >= c.hd) continue;
        uint2 codes = codes_of<E4M3>(values(x[i]), by);
        if (by == 0.0f) codes = make_uint2(0, 0);  // an infinity or a NaN in the row
        *reinterpret_cast<uint2*>((f < c.kv_heads ? c.k : c.v) + row_of(f) * c.hd + d) = codes;
    }
}

// ------------------------------------------------------------------------------------------------ read back
template <bool E4M3>
__device__ __forceinline__ F8 values_of(uint2 u, float s) {
    F8 r;
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (E4M3) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> (16 * j) & 0xffffu), __NV_E4M3));
                const float2 f = __half22float2(a);
                r.v[4 * i + 2 * j] = __fmul_rn(f.x, s);
                r.v[4 * i + 2 * j + 1] = __fmul_rn(f.y, s);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) r.v[4 * i + j] = __fmul_rn((float)(int8_t)(w[i] >> (8 * j) & 0xffu), s);
        }
    }
    return r;
}

// As the write: a warp takes kFlight heads a group from one token; a thread's one load at a time had taken 238 us for the 65537. `parts` = 2: keys and values, 1: the one whose rows are given.
constexpr int kFlight = 4;
template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256)
kv_read_kernel(KvView c, const int64_t* __restrict__ slots, int M, T* __restrict__ k, int64_t ldk, T* __restrict__ v, int64_t ldv,
               int parts, int warps_a_token) {
    constexpr int G = 32 / LANES;
    const int lane = threadIdx.x % LANES, g = (threadIdx.x & 31) / LANES, d = 8 * lane;
    const uint32_t w = blockIdx.x * 8u + (threadIdx.x >> 5), token = w / (uint32_t)warps_a_token;
    const int64_t m = token;
    const int f0 = (int)(w - token * (uint32_t)warps_a_token) * G + g, step = warps_a_token * G, heads = parts * c.kv_heads;
    griddep_wait();
    griddep_launch();
    if (m >= M || d >= c.hd) return;
    const int64_t slot = slots[m];
    const bool there = slot >= 0 && slot < c.n_pages << c.page_shift;
    if (slot >= 0 && !there && f0 == 0 && lane == 0) atomicOr(&g_device_error, kErrIndex);
    const int64_t row0 =
        there ? (((slot >> c.page_shift) * c.kv_heads) << c.page_shift) + (slot & ((1 << c.page_shift) - 1)) : 0;
    uint2 u[kFlight];
    float s[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
        const int f = f0 + i * step;
        u[i] = make_uint2(0, 0);
        s[i] = 0.0f;
        if (there && f < heads) {
            const bool is_v = !k || f >= c.kv_heads;
            const int64_t row = row0 + ((int64_t)(f >= c.kv_heads ? f - c.kv_heads : f) << c.page_shift);
            u[i] = *reinterpret_cast<const uint2*>((is_v ? c.v : c.k) + row * c.hd + d);
            s[i] = (is_v ? c.vs : c.ks)[row];
        }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
        const int f = f0 + i * step;
        if (f >= heads) break;
        const bool is_v = !k || f >= c.kv_heads;
        const int h = f >= c.kv_heads ? f - c.kv_heads : f;
        F8 x = values_of<E4M3>(u[i], s[i]);
        if (!there) x = F8{{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
        store8((is_v ? v + m * ldv : k + m * ldk) + (int64_t)h * c.hd + d, x);
    }
}

template <typename T>
cudaError_t rope_typed(const void* x, int64_t ldx, int64_t M, int n_heads, int hd, const int32_t* pos, int64_t ldpos,
                       const RopePairs& pairs, void* y, int64_t ldy, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    const bool wide = (hd / 2) % W == 0 && hd / 2 / W <= 32 &&
                      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0 && ldx % W == 0 && ldy % W == 0;
    if (!wide)
        return launch_pdl(rope_axes_any_kernel<T>, dim3((unsigned)ceil_div(M, kRopeRows)), dim3(256), st, static_cast<const T*>(x),
                          ldx, M, n_heads, hd, pos, ldpos, pairs, static_cast<T*>(y), ldy);
    // A warp takes all of a row's heads, which share its angles; with few rows, one step in flight of them.
    const int step = 32 / (hd / 2 / W) * kRopeFlight, per = M >= 16 * 148 || n_heads < step ? n_heads : step;
    const int warps = (int)ceil_div(n_heads, per);
    return launch_pdl(rope_axes_kernel<T, W>, dim3((unsigned)ceil_div(M * warps, 8)), dim3(256), st, static_cast<const T*>(x), ldx,
                      (int)M, n_heads, hd, pos, ldpos, pairs, static_cast<T*>(y), ldy, per, warps);
}

template <typename T, bool E4M3, int LANES>
cudaError_t write_typed(const KvView& c, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t M,
                        const int64_t* slots, cudaStream_t st) {
    const int per = (int)ceil_div(2 * c.kv_heads, kWriteSteps<LANES> * (32 / LANES));
    return launch_pdl(kv_write_kernel<T, E4M3, LANES>, dim3((unsigned)ceil_div(M * per, 8)), dim3(256), st, c,
                      static_cast<const T*>(k), ldk, static_cast<const T*>(v), ldv, (int)M, slots, per);
}
template <typename T, bool E4M3, int LANES>
cudaError_t read_typed(const KvView& c, const int64_t* slots, int64_t M, void* k, int64_t ldk, void* v, int64_t ldv,
                       cudaStream_t st) {
    const int parts = (k ? 1 : 0) + (v ? 1 : 0), per = (int)ceil_div(parts * c.kv_heads, kFlight * (32 / LANES));
    return launch_pdl(kv_read_kernel<T, E4M3, LANES>, dim3((unsigned)ceil_div(M * per, 8)), dim3(256), st, c, slots, (int)M,
                      static_cast<T*>(k), ldk, static_cast<T*>(v), ldv, parts, per);
}

// Lanes for a head of hd values, eight each: a power of two that divides a warp.
#define KV_LANES(fn, T, E, ...)                             \
    (c.hd > 64   ? fn<T, E, 16>(__VA_ARGS__)                \
     : c.hd > 32 ? fn<T, E, 8>(__VA_ARGS__)                 \
                 : fn<T, E, 4>(__VA_ARGS__))
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
