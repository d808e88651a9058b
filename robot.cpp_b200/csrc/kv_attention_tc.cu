// kv_attention_tc.cu -- attention of many query rows for each key/value head over the paged 8-bit cache, on the tcgen05
// tensor cores: prompts, chunks of long prompts, and a batch's rows on a shared prefix.
//
// Mathematics as in kv_attention.cu: the 8-bit codes are exact in fp16, a query row scaled by a power of two is one
// (bf16) or two (fp32) fp16 parts, and so are the probabilities times the value scale. One MMA a part:
//   S = sum over parts Q_part K^T,  O += sum over parts P_part V   (fp32 accumulation in tensor memory).
// Floor: 4 * pairs * hd operations a head times the parts, at the fp16 rate.
//
// A block holds 128 query rows (tokens x the heads of a group) of one sequence and key/value head and walks its keys in
// tiles of 128. Warps 8-11 bring codes from the pages to registers, unpack them and store fp16 tiles in the 128-byte
// swizzled layout that serves K as a K-major and V as an MN-major operand; warp 12 issues the MMAs; warps 0-7 hold two
// threads for each row (64 keys each) and do the softmax from tensor memory, writing P over S. Three S/P buffers: the
// scores of the next tile are computed while the softmax of this one runs.
// The running maximum is moved only when a tile exceeds it by 2^8, so the outputs in tensor memory are rarely rescaled.
//
// Every wait is bounded: after one that ran out the error word is set, further waits of the block return at once, no more
// MMAs are issued, those in flight are waited for, and tensor memory is freed.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "b2s_internal.h"
#include "kv_internal.h"

namespace b2s {

namespace kvt {
constexpr int kRows = 128, kKeys = 128;
constexpr int kSoftWarps = 8, kConvWarps = 4, kThreads = 32 * (kSoftWarps + kConvWarps + 1);
constexpr int kTmemCols = 512, kOcol = 384;  // S/P buffers at 0, 128, 256
constexpr int kBlock = kKeys * 128;          // bytes of 128 rows x 64 fp16 values
struct Misc {
    float ks[4][kKeys], vs[4][kKeys];  // scales of four tiles in flight
    int vexp[4][kConvWarps];           // largest value-scale exponent of each 32 keys
    uint32_t there[4][kConvWarps];     // keys that exist
    float red[2][2][2][kRows];         // [tile parity][maximum, largest value scale][half][row]
    float rf[kRows];                   // takes a row's scores back to log2 units
    uint64_t kfull[2], kfree[2], vfull[2], vfree[2], sfull[3], pfull[3], pvd[3], scfull[4], drain;
    int64_t scan[kSoftWarps + kConvWarps + 1];
    int64_t found[2];
    uint32_t tmem;
    int abort;
};
template <int HDP, int PARTS>
constexpr size_t kSmem = 1024 + (size_t)(HDP / 64) * kBlock * (PARTS + 4) + sizeof(Misc);
}  // namespace kvt

namespace {

using namespace kvt;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2_biased(int e) { return __int_as_float(e << 23); }
__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t w) {
    uint32_t d;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(d) : "r"(w));
    return d;
}
__device__ __forceinline__ uint32_t pack_h2(float x0, float x1) {
    const __half2 h = __floats2half2_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Four consecutive codes as two pairs of fp16. int8: 0x6400 | (b ^ 0x80) is 1152 + b; both steps are exact.
template <bool E4M3>
__device__ __forceinline__ void unpack4(uint32_t w, uint32_t& p0, uint32_t& p1) {
    if (E4M3) {
        p0 = e4m3x2_to_h2(w);
        p1 = e4m3x2_to_h2(w >> 16);
    } else {
        p0 = sub_h2((__byte_perm(w, 0, 0x4140) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
        p1 = sub_h2((__byte_perm(w, 0, 0x4342) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    }
}

// V as an MN-major operand with 128-byte swizzle: 64 values of hd are 128 bytes, 8 keys make an atom (stride 1024), the
// next 64 values lie kBlock bytes on.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(kBlock >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// kind::f16: D f32, A and B fp16; B's major-ness in bit 16.
constexpr uint32_t idesc_f16(int N, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Paired fp32 operations (each lane an IEEE operation).
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unf2(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

struct Rows {
    int lo, n, len, tiles;  // first query row, query rows, keys, blocks of 128 (token, head of group) rows
};
__device__ __forceinline__ Rows rows_of(const KvAttnArgs& a, int b) {
    Rows s;
    const int lo = a.q_start[b * a.q_stride], hi = a.q_start[(b + 1) * a.q_stride];
    int64_t len = a.kv_len ? (int64_t)a.kv_len[b] : a.kv_const;
    const int64_t cap = a.max_pages << a.c.page_shift;
    bool bad = lo < 0 || hi < lo || hi > a.M;
    s.lo = lo;
    s.n = bad ? 0 : hi - lo;
    if (len < 0 || len > cap) {
        bad = true;
        len = len < 0 ? 0 : cap;
    }
    if (bad) atomicOr(&g_device_error, kErrIndex);
    s.len = (int)len;
    s.tiles = s.n * a.group > a.min_rows ? (s.n * a.group + kRows - 1) / kRows : 0;
    return s;
}

// A wait that ends: at its phase, after kWaitLimitNs, or at once when another wait of the block ran out.
__device__ __forceinline__ bool wait(Misc* ms, uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    volatile int* ab = &ms->abort;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*ab) return false;
        if ((i & 15u) == 15u && global_timer_ns() - t0 > kWaitLimitNs) break;
    }
    *ab = 1;
    atomicOr(&g_device_error, 1u);
    return false;
}

template <int HDP, bool E4M3, int PARTS>
__global__ void __launch_bounds__(kThreads, 1) kv_attention_tc_kernel(const KvAttnArgs a, int units, int splits) {
    constexpr int kTileBytes = HDP / 64 * kBlock;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sK = sQ + PARTS * kTileBytes;
    uint8_t* sV = sK + 2 * kTileBytes;
    Misc* ms = reinterpret_cast<Misc*>(sV + 2 * kTileBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    griddep_launch();

    // ---- which sequence, row block, head and share of the keys: later row blocks, which see more keys, go first
    const int h = blockIdx.x % a.c.kv_heads;
    const int64_t rest = blockIdx.x / a.c.kv_heads;
    const int split = (int)(rest / units);
    int unit = (int)(rest - (int64_t)split * units);
    {
        int64_t total = 0, w = 0, incl = 0;
        for (int pass = 0; pass < 2; ++pass) {  // the total first: the order is from the last row block
            int64_t before = 0;
            for (int base = 0; base < a.batch; base += kThreads) {
                const int b = base + tid;
                w = b < a.batch ? rows_of(a, b).tiles : 0;
                int64_t v = w;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += u;
                }
                __syncthreads();
                if (lane == 31) ms->scan[warp] = v;
                __syncthreads();
                int64_t sum = 0;
                for (int i = 0; i < kThreads / 32; ++i) {
                    if (i < warp) v += ms->scan[i];
                    sum += ms->scan[i];
                }
                incl = v + before;
                before += sum;
                if (pass == 1 && unit >= incl - w && unit < incl) {
                    ms->found[0] = b;
                    ms->found[1] = unit - (incl - w);
                }
            }
            if (pass == 0) {
                total = before;
                if (unit >= total) return;  // the grid is sized by a bound
                unit = (int)(total - 1 - unit);
            }
        }
        __syncthreads();
    }
    const int b = (int)ms->found[0], row0 = (int)ms->found[1] * kRows;
    const Rows sq = rows_of(a, b);
    const int rows = min(kRows, sq.n * a.group - row0);
    // keys that the last row sees
    const int most = a.causal ? min(sq.len, max(0, sq.len - sq.n + (row0 + rows - 1) / a.group + 1)) : sq.len;
    const int all_tiles = (most + kKeys - 1) / kKeys;
    const int t0 = (int)((int64_t)all_tiles * split / splits), nt = (int)((int64_t)all_tiles * (split + 1) / splits) - t0;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ms->kfull[i], 32 * kConvWarps);
            mbar_init(&ms->vfull[i], 32 * kConvWarps);
            mbar_init(&ms->kfree[i], 1);
            mbar_init(&ms->vfree[i], 1);
        }
        for (int i = 0; i < 3; ++i) {
            mbar_init(&ms->sfull[i], 1);
            mbar_init(&ms->pfull[i], 32 * kSoftWarps);
            mbar_init(&ms->pvd[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&ms->scfull[i], 32 * kConvWarps);
        mbar_init(&ms->drain, 1);
        ms->abort = 0;
        fence_mbar_init();
    }
    if (warp == kSoftWarps + kConvWarps) {
        tmem_alloc(&ms->tmem, kTmemCols);
        tmem_relinquish();
    }
    // ---- the query rows: a warp takes a row at a time, four values a lane
    const bool negative = a.scale_log2e < 0.0f, zero = a.scale_log2e == 0.0f;
    if (warp < kSoftWarps) {
        const int d = 4 * lane;
#pragma unroll 4
        for (int r = warp; r < kRows; r += kSoftWarps) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows && d < a.c.hd && !zero) {
                const int i = (row0 + r) / a.group, head = h * a.group + (row0 + r - i * a.group);
                const int64_t at = (sq.lo + (int64_t)i) * a.ldq + (int64_t)head * a.c.hd + d;
                if (a.bf16) {
                    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.q) + at);
                    x = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                                    __uint_as_float(u.y & 0xffff0000u));
                } else {
                    x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at);
                }
            }
            float big = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
            big = warp_max(big);
            const int up = min(253, 268 - (__float_as_int(big) >> 23));  // the largest element goes to [2^14, 2^15)
            const float mul = negative ? -pow2_biased(up) : pow2_biased(up);
            if (lane == 0) ms->rf[r] = zero ? 1.0f : fmaxf(__fmul_rn(pow2_biased(254 - up), fabsf(a.scale_log2e)), 0x1p-126f);
            const float y[4] = {__fmul_rn(x.x, mul), __fmul_rn(x.y, mul), __fmul_rn(x.z, mul), __fmul_rn(x.w, mul)};
            if (d < HDP) {
                uint8_t* p = sQ + (d >> 6) * kBlock + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 4) * 2;
                const uint2 hi = make_uint2(pack_h2(y[0], y[1]), pack_h2(y[2], y[3]));
                *reinterpret_cast<uint2*>(p) = hi;
                if (PARTS == 2) {
                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
                    const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                    *reinterpret_cast<uint2*>(p + kTileBytes) = make_uint2(
                        pack_h2(__fsub_rn(y[0], f0.x), __fsub_rn(y[1], f0.y)), pack_h2(__fsub_rn(y[2], f1.x), __fsub_rn(y[3], f1.y)));
                }
            }
        }
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ms->tmem;

    if (warp >= kSoftWarps && warp < kSoftWarps + kConvWarps) {
        // ================================================================ codes to fp16 tiles
        constexpr int kChunks = HDP / 16, kPer = kChunks;  // 16-byte code chunks of a row; chunks of a thread per tile
        constexpr int kRowsPer = 32 / kChunks;             // rows that a warp covers at once
        const int cw = warp - kSoftWarps, c = lane % kChunks, rsub = lane / kChunks;
        const int mask = (1 << a.c.page_shift) - 1;
        const int32_t* pg = a.pages + (int64_t)b * a.ld_pages;
        const bool on_c = c * 16 < a.c.hd;
        // a warp's 32 keys of a tile lie in at most two pages: those of its first and its 17th key
        int pa = 0, pb = 0;
        auto fetch = [&](int j) {
            const int k0 = (t0 + j) * kKeys + cw * 32;
            pa = k0 < sq.len ? pg[k0 >> a.c.page_shift] : 0;
            pb = k0 + 16 < sq.len ? pg[(k0 + 16) >> a.c.page_shift] : 0;
        };
        int64_t ra = 0, rb = 0;
        int k0 = 0;
        bool ok_a = false, ok_b = false;
        auto place = [&](int j) {
            k0 = (t0 + j) * kKeys + cw * 32;
            ok_a = pa >= 0 && pa < a.c.n_pages;
            ok_b = pb >= 0 && pb < a.c.n_pages;
            if (!(ok_a && ok_b) && lane == 0) atomicOr(&g_device_error, kErrIndex);
            ra = (((int64_t)pa * a.c.kv_heads + h) << a.c.page_shift) + (k0 & mask);
            rb = (((int64_t)pb * a.c.kv_heads + h) << a.c.page_shift) + ((k0 + 16) & mask) - 16;
        };
        uint4 kr[kPer], vr[kPer];
        float ksc = 0.0f, vsc = 0.0f;
        bool here = false;
        auto load = [&](const uint8_t* base, uint4 (&r)[kPer]) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int row = i * kRowsPer + rsub;
                r[i] = make_uint4(0, 0, 0, 0);
                if ((row < 16 ? ok_a : ok_b) && k0 + row < sq.len && on_c)
                    r[i] = __ldg(reinterpret_cast<const uint4*>(base + ((row < 16 ? ra : rb) + row) * a.c.hd + c * 16));
            }
        };
        auto load_scales = [&]() {
            here = (lane < 16 ? ok_a : ok_b) && k0 + lane < sq.len;
            ksc = vsc = 0.0f;
            if (here) {
                const int64_t row = (lane < 16 ? ra : rb) + lane;
                ksc = __ldg(a.c.ks + row);
                vsc = __ldg(a.c.vs + row);
            }
        };
        auto store = [&](uint8_t* tile, const uint4 (&r)[kPer]) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int row = cw * 32 + i * kRowsPer + rsub;
                uint32_t w[8];
                unpack4<E4M3>(r[i].x, w[0], w[1]);
                unpack4<E4M3>(r[i].y, w[2], w[3]);
                unpack4<E4M3>(r[i].z, w[4], w[5]);
                unpack4<E4M3>(r[i].w, w[6], w[7]);
                uint8_t* p = tile + (c >> 2) * kBlock + row * 128;
                const int ch = 2 * (c & 3), sw = (c >> 2) & 1;  // the second block's lanes store their halves in turn
                const uint4 x0 = make_uint4(w[0], w[1], w[2], w[3]), x1 = make_uint4(w[4], w[5], w[6], w[7]);
                *reinterpret_cast<uint4*>(p + (((ch + sw) ^ (row & 7)) << 4)) = sw ? x1 : x0;
                *reinterpret_cast<uint4*>(p + (((ch + 1 - sw) ^ (row & 7)) << 4)) = sw ? x0 : x1;
            }
        };
        if (nt > 0) {
            fetch(0);
            place(0);
            load(a.c.k, kr);
            load_scales();
            if (nt > 1) fetch(1);
        }
        for (int j = 0; j < nt; ++j) {
            const int st = j & 1;
            load(a.c.v, vr);  // this tile's places are still set
            if (j >= 2) wait(ms, &ms->kfree[st], (uint32_t)((j >> 1) - 1) & 1u);
            store(sK + st * kTileBytes, kr);
            fence_proxy_async_smem();
            mbar_arrive(&ms->kfull[st]);
            ms->ks[j & 3][cw * 32 + lane] = ksc;
            ms->vs[j & 3][cw * 32 + lane] = vsc;
            const int e = __reduce_max_sync(0xffffffffu, here ? (__float_as_int(fabsf(vsc)) >> 23) : 0);
            const uint32_t bits = __ballot_sync(0xffffffffu, here);
            if (lane == 0) {
                ms->vexp[j & 3][cw] = e;
                ms->there[j & 3][cw] = bits;
            }
            __syncwarp();
            mbar_arrive(&ms->scfull[j & 3]);
            if (j + 1 < nt) {
                place(j + 1);
                load(a.c.k, kr);
                load_scales();
                if (j + 2 < nt) fetch(j + 2);
            }
            if (j >= 2) wait(ms, &ms->vfree[st], (uint32_t)((j >> 1) - 1) & 1u);
            store(sV + st * kTileBytes, vr);
            fence_proxy_async_smem();
            mbar_arrive(&ms->vfull[st]);
        }
    } else if (warp == kSoftWarps + kConvWarps) {
        // ================================================================ MMAs
        if (lane == 0) {
            constexpr uint32_t kIdS = idesc_f16(kKeys, false), kIdO = idesc_f16(HDP, true);
            const uint32_t q0 = smem_u32(sQ), k0 = smem_u32(sK), v0 = smem_u32(sV);
            bool ok = true;
            auto scores = [&](int j) {
                ok = wait(ms, &ms->kfull[j & 1], (uint32_t)(j >> 1) & 1u) && ok;
                // the buffer's last reader, the product with the probabilities of tile j - 3, has to be through
                if (j >= 3) ok = wait(ms, &ms->pvd[j % 3], (uint32_t)(j / 3 - 1) & 1u) && ok;
                if (!ok) return;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(j % 3) * kKeys, kt = k0 + (j & 1) * kTileBytes;
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int s = 0; s < HDP / 16; ++s) {
                        const uint32_t off = (s >> 2) * kBlock + (s & 3) * 32;
                        mma_ss(d, umma_desc_k_sw128(q0 + part * kTileBytes + off), umma_desc_k_sw128(kt + off), kIdS,
                               (part > 0 || s > 0) ? 1u : 0u);
                    }
                tc_commit(&ms->sfull[j % 3]);
                tc_commit(&ms->kfree[j & 1]);
            };
            if (nt > 0) scores(0);
            for (int j = 0; j < nt; ++j) {
                if (j + 1 < nt) scores(j + 1);
                ok = wait(ms, &ms->vfull[j & 1], (uint32_t)(j >> 1) & 1u) && ok;
                ok = wait(ms, &ms->pfull[j % 3], (uint32_t)(j / 3) & 1u) && ok;
                if (!ok) continue;
                tc_fence_after();
                const uint32_t p = tmem + (uint32_t)(j % 3) * kKeys, vt = v0 + (j & 1) * kTileBytes;
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int s = 0; s < kKeys / 16; ++s)
                        mma_ts(tmem + kOcol, p + part * 64 + s * 8, desc_mn_sw128(vt + s * 2048), kIdO,
                               (j > 0 || part > 0 || s > 0) ? 1u : 0u);
                tc_commit(&ms->pvd[j % 3]);
                tc_commit(&ms->vfree[j & 1]);
            }
            if (!ok) {  // let what was issued finish before tensor memory is freed
                tc_commit(&ms->drain);
                mbar_wait(&ms->drain, 0, 2u);
            }
        }
        __syncwarp();
    } else {
        // ================================================================ softmax
        const int quad = warp & 3, half = warp >> 2, r = quad * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
        const bool mine = r < rows;
        const int tok = (row0 + r) / a.group;
        // a row that is not there never masks (its results are dropped)
        const int limit = !mine ? 0x7fffffff : a.causal ? sq.len - sq.n + tok + 1 : sq.len;
        const int wmin = __reduce_min_sync(0xffffffffu, limit);
        const float rf = ms->rf[r];
        float m = -INFINITY, l = 0.0f;
        int vref = 8;
        for (int j = 0; j < nt; ++j) {
            const int key0 = (t0 + j) * kKeys + half * 64;
            wait(ms, &ms->scfull[j & 3], (uint32_t)(j >> 2) & 1u);
            const uint32_t w0 = ms->there[j & 3][2 * half], w1 = ms->there[j & 3][2 * half + 1];
            const uint32_t wo = ms->there[j & 3][2 - 2 * half] & ms->there[j & 3][3 - 2 * half];
            const bool masked = (w0 & w1 & wo) != 0xffffffffu || (t0 + j + 1) * kKeys > wmin;
            const float4* ksp = reinterpret_cast<const float4*>(&ms->ks[j & 3][half * 64]);
            const float4* vsp = reinterpret_cast<const float4*>(&ms->vs[j & 3][half * 64]);
            int e = max(max(ms->vexp[j & 3][0], ms->vexp[j & 3][1]), max(ms->vexp[j & 3][2], ms->vexp[j & 3][3]));
            wait(ms, &ms->sfull[j % 3], (uint32_t)(j / 3) & 1u);
            tc_fence_after();
            const uint32_t sbuf = lane_addr + (uint32_t)(j % 3) * kKeys;
            float s[64];
            {
                uint32_t x[32], y[32];
                tmem_ld_32x32b_x32(sbuf + half * 64, x);
                tmem_ld_32x32b_x32(sbuf + half * 64 + 32, y);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    s[i] = __uint_as_float(x[i]);
                    s[32 + i] = __uint_as_float(y[i]);
                }
            }
            float mx = -INFINITY, vmx = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float4 f = ksp[i];
                unf2(mul2(f2(s[4 * i], s[4 * i + 1]), f2(f.x, f.y)), s[4 * i], s[4 * i + 1]);
                unf2(mul2(f2(s[4 * i + 2], s[4 * i + 3]), f2(f.z, f.w)), s[4 * i + 2], s[4 * i + 3]);
            }
            uint32_t see0 = 0xffffffffu, see1 = 0xffffffffu;  // keys of this thread that the row sees
            if (masked) {
                const int left = limit - key0;
                see0 = w0 & (left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u);
                see1 = w1 & (left >= 64 ? 0xffffffffu : left > 32 ? (1u << (left - 32)) - 1u : 0u);
                const float* vp = &ms->vs[j & 3][half * 64];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (!((see0 >> i) & 1)) s[i] = -INFINITY; else vmx = fmaxf(vmx, fabsf(vp[i]));
                    if (!((see1 >> i) & 1)) s[32 + i] = -INFINITY; else vmx = fmaxf(vmx, fabsf(vp[32 + i]));
                }
            }
#pragma unroll
            for (int i = 0; i < 64; ++i) mx = fmaxf(mx, s[i]);
            // ---- the row's two threads: from here on S is in registers, and P may be written over it
            ms->red[j & 1][0][half][r] = mx;
            if (masked) ms->red[j & 1][1][half][r] = vmx;
            tc_fence_before();
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
            tc_fence_after();
            mx = fmaxf(mx, ms->red[j & 1][0][half ^ 1][r]);
            if (masked) e = __float_as_int(fmaxf(vmx, ms->red[j & 1][1][half ^ 1][r])) >> 23;
            const float mt = __fmul_rn(mx, rf);
            const bool move = mt > __fadd_rn(m, 8.0f) || (m == -INFINITY && mt > -INFINITY) || e >= vref;
            if (__any_sync(0xffffffffu, move)) {
                float f = 1.0f;
                if (move) {
                    const float mn = fmaxf(m, mt);
                    f = m == -INFINITY ? 0.0f : ex2(__fsub_rn(m, mn));
                    l = __fmul_rn(l, f);
                    m = mn;
                    const int nref = e >= vref ? min(e + 2, 255) : vref;
                    f = nref - vref > 126 ? 0.0f : __fmul_rn(f, pow2_biased(127 - (nref - vref)));
                    vref = nref;
                }
                if (j > 0) {
                    wait(ms, &ms->pvd[(j - 1) % 3], (uint32_t)((j - 1) / 3) & 1u);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < HDP / 2; c += 16) {
                        const uint32_t at = lane_addr + kOcol + half * (HDP / 2) + c;
                        uint32_t x[16];
                        tmem_ld_x16(at, x);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__fmul_rn(__uint_as_float(x[i]), f));
                        tmem_st_x16(at, x);
                    }
                }
            }
            const float mu = m == -INFINITY ? 0.0f : -m, vmul = pow2_biased(260 - vref);
            const F2 rf2 = f2(rf, rf), mu2 = f2(mu, mu), vmul2 = f2(vmul, vmul);
            F2 l2 = f2(0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 f = vsp[q * 8 + i];
                    float fv[4] = {f.x, f.y, f.z, f.w};
                    if (masked) {  // a value scale that the row does not see may be anything
                        const uint32_t see = (q ? see1 : see0) >> (4 * i);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (!((see >> k) & 1)) fv[k] = 0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int at = q * 32 + 4 * i + 2 * k;
                        float x0, x1;
                        unf2(fma2(f2(s[at], s[at + 1]), rf2, mu2), x0, x1);
                        const F2 p = f2(ex2(x0), ex2(x1));
                        l2 = add2(l2, p);
                        unf2(mul2(p, mul2(f2(fv[2 * k], fv[2 * k + 1]), vmul2)), x0, x1);
                        hi[2 * i + k] = pack_h2(x0, x1);
                        if (PARTS == 2) {
                            const float2 b2 = __half22float2(*reinterpret_cast<const __half2*>(&hi[2 * i + k]));
                            lo[2 * i + k] = pack_h2(__fsub_rn(x0, b2.x), __fsub_rn(x1, b2.y));
                        }
                    }
                }
                tmem_st_x16(sbuf + half * 32 + q * 16, hi);
                if (PARTS == 2) tmem_st_x16(sbuf + 64 + half * 32 + q * 16, lo);
            }
            float la, lb;
            unf2(l2, la, lb);
            l = __fadd_rn(l, __fadd_rn(la, lb));
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&ms->pfull[j % 3]);
        }
        // ---- the row's sum, and the outputs: each of its two threads writes half of the columns
        ms->red[nt & 1][0][half][r] = l;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
        l = __fadd_rn(ms->red[nt & 1][0][0][r], ms->red[nt & 1][0][1][r]);
        if (nt > 0) {
            wait(ms, &ms->pvd[(nt - 1) % 3], (uint32_t)((nt - 1) / 3) & 1u);
            tc_fence_after();
        }
        const float back = pow2_biased(vref - 6);
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        const int64_t grow = sq.lo + (int64_t)tok;
        const int head = h * a.group + (row0 + r - tok * a.group);
        const int64_t si = ((int64_t)split * a.M + grow) * a.heads + head;
        if (a.to_state && mine && half == 0) {
            a.out.m[si] = m;
            a.out.l[si] = l;
        }
#pragma unroll
        for (int c = 0; c < HDP / 2; c += 16) {
            uint32_t x[16];
            if (nt > 0) {
                tmem_ld_x16(lane_addr + kOcol + half * (HDP / 2) + c, x);
                tc_wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = 0;
            }
            const int d = half * (HDP / 2) + c;
            if (!mine || d >= a.c.hd) continue;
            float o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __fmul_rn(__uint_as_float(x[i]), back);
            if (a.to_state) {
                float4* p = reinterpret_cast<float4*>(a.out.o + si * a.c.hd + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = l == 0.0f ? 0.0f : __fmul_rn(o[i], inv);
            const int64_t at = grow * a.ldo + (int64_t)head * a.c.hd + d;
            if (a.bf16) {
                uint4* p = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o) + at);
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const __nv_bfloat162 y = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t*>(&y);
                }
                p[0] = make_uint4(w[0], w[1], w[2], w[3]);
                p[1] = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
                float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.o) + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSoftWarps + kConvWarps) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---------------------------------------------------------------- joining pieces
// One warp for each (row of q, head): the pieces of this pass and the added ones, in that order, then the output row.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) kv_state_join_kernel(const KvAttnArgs a) {
    const int lane = threadIdx.x & 31, d = 4 * lane;
    griddep_wait();
    griddep_launch();
    const int64_t n = a.M * a.heads;
    for (int64_t i = (int64_t)blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5); i < n; i += (int64_t)gridDim.x * (kJoinThreads / 32)) {
        const int64_t row = i / a.heads;
        const int head = (int)(i - row * a.heads);
        // the row's sequence: the last one that does not start behind it, 32 candidates a step
        int lo = 0, count = a.batch;
        while (count > 0) {
            const int step = (count + 31) / 32, at = lo + lane * step;
            const bool before = at < lo + count && a.q_start[at * a.q_stride] <= row;
            const int k = 32 - __clz(__ballot_sync(0xffffffffu, before));  // candidates that start at or before the row
            if (k == 0) {
                count = 0;
                lo = -1;
            } else {
                const int first = lo + (k - 1) * step;
                count = min(step, lo + count - first);
                lo = first;
                if (step == 1) break;
            }
        }
        if (lo < 0) continue;
        const Rows sq = rows_of(a, lo);
        if (sq.tiles == 0 || row >= sq.lo + (int64_t)sq.n) continue;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const int pieces = a.out.pieces + a.add.pieces;
        for (int s = 0; s < pieces; ++s) {
            const bool own = s < a.out.pieces;
            const AttnState& st = own ? a.out : a.add;
            const int64_t at = (int64_t)(own ? s : s - a.out.pieces) * n + i;
            const float mi = st.m[at], li = st.l[at], mn = fmaxf(m, mi);
            const float x = m == -INFINITY ? 0.0f : ex2(__fsub_rn(m, mn)), y = mi == -INFINITY ? 0.0f : ex2(__fsub_rn(mi, mn));
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (d < a.c.hd) v = *reinterpret_cast<const float4*>(st.o + at * a.c.hd + d);
            l = __fmaf_rn(l, x, __fmul_rn(li, y));
            o.x = __fmaf_rn(o.x, x, __fmul_rn(v.x, y));
            o.y = __fmaf_rn(o.y, x, __fmul_rn(v.y, y));
            o.z = __fmaf_rn(o.z, x, __fmul_rn(v.z, y));
            o.w = __fmaf_rn(o.w, x, __fmul_rn(v.w, y));
            m = mn;
        }
        if (d >= a.c.hd) continue;
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        o = l == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f)
                      : make_float4(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv), __fmul_rn(o.z, inv), __fmul_rn(o.w, inv));
        const int64_t at = row * a.ldo + (int64_t)head * a.c.hd + d;
        if (a.bf16) {
            const __nv_bfloat162 y0 = __floats2bfloat162_rn(o.x, o.y), y1 = __floats2bfloat162_rn(o.z, o.w);
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.o) + at) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&y0), *reinterpret_cast<const uint32_t*>(&y1));
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = o;
        }
    }
}

template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), int64_t grid, int block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int HDP, bool E4M3, int PARTS>
cudaError_t launch_typed(const KvAttnArgs& a, int64_t units, int splits, cudaStream_t st) {
    auto kernel = kv_attention_tc_kernel<HDP, E4M3, PARTS>;
    const size_t smem = kSmem<HDP, PARTS>;
    const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, units * a.c.kv_heads * splits, kThreads, smem, st, a, (int)units, splits);
}

}  // namespace

int64_t kv_attn_tc_units(int64_t M, int batch, int group) { return M * group / kRows + batch; }

cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, int splits, cudaStream_t st) {
    if (a.batch <= 0 || a.M <= 0) return cudaSuccess;
    const int64_t units = kv_attn_tc_units(a.M, a.batch, a.group);
    if (a.c.hd > 64) {
        if (a.bf16) return a.c.e4m3 ? launch_typed<128, true, 1>(a, units, splits, st) : launch_typed<128, false, 1>(a, units, splits, st);
        return a.c.e4m3 ? launch_typed<128, true, 2>(a, units, splits, st) : launch_typed<128, false, 2>(a, units, splits, st);
    }
    if (a.bf16) return a.c.e4m3 ? launch_typed<64, true, 1>(a, units, splits, st) : launch_typed<64, false, 1>(a, units, splits, st);
    return a.c.e4m3 ? launch_typed<64, true, 2>(a, units, splits, st) : launch_typed<64, false, 2>(a, units, splits, st);
}

cudaError_t launch_kv_state_join(const KvAttnArgs& a, cudaStream_t st) {
    const int64_t blocks = ceil_div(a.M * a.heads, kJoinThreads / 32);
    return launch_pdl(kv_state_join_kernel, blocks < 148 * 8 ? blocks : 148 * 8, kJoinThreads, 0, st, a);
}

}  // namespace b2s
