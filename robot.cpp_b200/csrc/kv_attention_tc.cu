// kv_attention_tc.cu -- attention of many query rows for each key/value head over the paged 8-bit cache, on the tcgen05
// tensor cores: prompts, chunks of long prompts, and a batch's rows on a shared prefix.
//
// Mathematics as in kv_attention.cu: the 8-bit codes are exact in fp16; query rows scaled by a power of two are one
// (bf16) or two (fp32) fp16 parts, and the probabilities times the value scale are two. One MMA a part:
//   S = sum over parts Q_part K^T,  O += sum over parts P_part V   (fp32 accumulation in tensor memory).
// One part of P would round each weight to 2^-11: 2 to 5% of bf16 outputs then came out a step off (a chunk of 2048 tokens on
// 8192 took 572 us with it and takes 702 with two).
// Floor: 2 * pairs * hd operations a head for each part of Q and P, at the fp16 rate; next to it the exponentials, 16 a clock
// and SM.
//
// A block takes rows (tokens x the heads of a group) of one sequence and key/value head and walks its keys in tiles of 128.
// Four warps bring codes from the pages, unpack them and store fp16 tiles in the 128-byte swizzled layout that serves K as a
// K-major and V as an MN-major operand. Two groups of eight warps do the softmax from tensor memory, one thread for each row
// and half of a tile's keys, and write P over S. The groups are
//   PAIR: two blocks of 128 rows that share every unpacked tile (bf16, where unpacking would weigh as much as the products);
//   else: the even and the odd key tiles of the same 128 rows, each with its own reference, sum and outputs, joined at the
//         end (fp32, whose two-part queries leave no room for more rows; and bf16 calls that have no more).
// A group's two halves are streams of their own: 128 threads, 64 columns of S and P, one thread that issues the stream's MMAs.
// A stream's chain (scores, exponentials, outputs, the next scores over its P) has four others' work beside it: with one
// chain a group the tensor cores and the exponentials waited for each other (a pair of tiles took 7500 clocks, of which the
// products are 2048 and the exponentials 2048). Sixteen warps also because one warp a scheduler needs 570 clocks for 32 keys'
// exponentials and four need 280 each (measured alone; the special-function unit's own limit is 256).
// The reference of the exponentials is a whole number that moves only when probabilities grow past 2^5: sums and outputs are
// then multiplied by a power of two, which is exact, and the half tile's probabilities too, which keep what their two parts can
// hold. So scores are read once and no maximum is formed: 32 probabilities whose sum is at most 2^5, which those at or below
// their reference never pass, are each at most that, and only a larger sum asks for their maximum. (With 2^8 the references
// move less and fp32 chunks took 4% less time, but probabilities have four bits fewer above the end of fp16.) A row's outputs
// have one reference; its two streams commit their products to it in turn, and whoever finds the other's reference changed
// brings its own probabilities, or the outputs, under the larger one.
//
// Measured: 2 x up to 2048 bf16 tokens on 8192 e4m3 ones, causal, 32 heads on 8 of 128: 702 us, 506 TFLOP/s of the 1640 that a
// library product reaches (759 with P's second part counted); 1024 tokens on 4096 with 20 heads on 5: 148 us (fp32, whose Q has
// two parts too, 197 us). A stream's chain for 64 keys bounds it, no unit does, and tensor memory has no columns for more
// streams. A block of few tiles is mostly start (10,000 clocks: lengths, pages, Q, the first codes) and end (6,000): 8 prompts of
// 288 fp32 tokens take 59 us.
//
// Every wait is bounded: after one that ran out the error word is set, further waits of the block return at once, no more
// MMAs are issued, those in flight are waited for, and tensor memory is freed.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "b2s_internal.h"
#include "kv_internal.h"

namespace b2s {

namespace kvt {
constexpr int kRows = 128, kKeys = 128;
constexpr int kSoftWarps = 16, kConvWarps = 4, kThreads = 32 * (kSoftWarps + kConvWarps);
constexpr int kHalf = kKeys / 2;
constexpr int kTmemCols = 512, kOcol = 256;  // S/P of the four streams at 0, 64, 128, 192, O of the two groups at 256 and 384
constexpr int kBlock = kKeys * 128;          // bytes of 128 rows x 64 fp16 values
struct Rows {
    int lo, n, len, rows;  // first query row, query rows, keys, (token, head of group) rows that this pass takes
};
constexpr int kWide = 0x1000;
struct Misc {
    float ks[4][kKeys];        // key scales of four tiles in flight, times the factor that takes scores to log2 units
    float vs[4][kKeys];        // value scales
    float vn[4][kKeys];        // value scales over the power of two above the largest finite one of their 32 keys
    // [half] keys that exist of its two times 32, and that scale's biased exponents, 1..252, with kWide where scores may pass 2^24
    struct alignas(16) {
        uint32_t there[2];
        int vexp[2];
    } of[4][2];
    float om[2][kRows];        // [group][row] reference of the row's outputs: of the exponentials,
    int ov[2][kRows];          // and of the value scales
    float l[2][2][kRows];      // [group][half of the row's keys][row]
    uint64_t qfull, kfull[2], kfree[2], vfull[2], vfree[2], sfull[4], pvd[4], mpost[4], scfull[4], drain[4];
    int64_t scan[kThreads / 32];
    int64_t found[2];
    Rows seq;                  // that sequence
    float big[kSoftWarps];     // largest finite element of the warp's query rows
    uint32_t row_big[2 * kRows];  // the largest magnitude of each row, as bits
    uint32_t tmem;
    int abort;
};
template <int HDP, int PARTS, bool PAIR>
constexpr size_t kSmem = 1024 + (size_t)(HDP / 64) * kBlock * (PARTS * (PAIR ? 2 : 1) + 4) + kKeys * HDP + sizeof(Misc);
static_assert(kSmem<128, 2, false> <= 232448 && kSmem<128, 1, true> <= 232448, "shared memory");
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
// Four consecutive codes as two pairs of fp16: e4m3 (0, 1) and (2, 3), int8 (0, 2) and (1, 3), which saves it a byte
// permutation; queries are stored in that order too, and outputs are taken out of it. int8: 0x6400 | (b ^ 0x80) is 1152 + b;
// both steps are exact.
template <bool E4M3>
__device__ __forceinline__ void unpack4(uint32_t w, uint32_t& p0, uint32_t& p1) {
    if (E4M3) {
        p0 = e4m3x2_to_h2(w);
        p1 = e4m3x2_to_h2(w >> 16);
    } else {
        p0 = sub_h2((w & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
        p1 = sub_h2(((w >> 8) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    const int n = on ? 16 : 0;  // 0 bytes: nothing is read, zeros are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint4 x) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
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
// The MMAs and their commits are issued by one elected lane of a warp whose lanes all get here with the same operands: those
// then live in uniform registers. (Under a branch on the lane every operand is moved there one by one: 150 clocks an MMA
// where the tensor core needs 64.)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void commit_elected(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Loads from tensor memory are complete behind this; the operands keep their uses behind it.
__device__ __forceinline__ void wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28])
                 :
                 : "memory");
    asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) : : "memory");
}

__device__ __forceinline__ void wait_ld(uint32_t (&r)[8], uint32_t (&s)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(s[0]),
                   "+r"(s[1]), "+r"(s[2]), "+r"(s[3]), "+r"(s[4]), "+r"(s[5]), "+r"(s[6]), "+r"(s[7])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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
__device__ __forceinline__ F2 f2u(uint32_t a, uint32_t b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
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

__device__ __forceinline__ Rows rows_of(const KvAttnArgs& a, int b) {
    Rows s;
    int lo = a.q_start[b * a.q_stride], hi = a.q_start[(b + 1) * a.q_stride];
    if (!a.kv_len) {  // a shared prefix: every row that a sequence in range can have gets its state
        lo = 0;
        hi = rows_used(a, hi);
    }
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
    s.rows = s.n * a.group > a.min_rows ? s.n * a.group : 0;
    return s;
}

// A wait that ends: at its phase, after kWaitLimitNs, or at once when another wait of the block ran out. The thread is
// suspended for up to the hinted time at each try.
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(100000)
        : "memory");
    return ok != 0;
}
__device__ __noinline__ void wait_on(int* abort, uint64_t* bar, uint32_t parity) {
    volatile int* ab = abort;
    const uint64_t t0 = global_timer_ns();
    do {
        if (*ab || try_wait(bar, parity)) return;
    } while (global_timer_ns() - t0 <= kWaitLimitNs);
    *ab = 1;
    atomicOr(&g_device_error, 1u);
}
__device__ __forceinline__ void wait(Misc* ms, uint64_t* bar, uint32_t parity) {
    if (!try_wait(bar, parity)) wait_on(&ms->abort, bar, parity);
}

template <int HDP, bool E4M3, int PARTS, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) kv_attention_tc_kernel(const KvAttnArgs a, int units, int splits) {
    constexpr int kTileBytes = HDP / 64 * kBlock;
    constexpr int kBlkRows = PAIR ? 2 * kRows : kRows;  // rows of a block
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sK = sQ + PARTS * (PAIR ? 2 : 1) * kTileBytes;
    uint8_t* sV = sK + 2 * kTileBytes;
    uint8_t* raw = sV + 2 * kTileBytes;  // the next value tile's codes
    Misc* ms = reinterpret_cast<Misc*>(raw + kKeys * HDP);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // warp: the same in every lane
    griddep_wait();

    // ---- which sequence, row block, head and share of the keys: later row blocks, which see more keys, go first
    const int h = blockIdx.x % a.c.kv_heads;
    const int rest = blockIdx.x / a.c.kv_heads, split = rest / units;
    int unit = rest - split * units;
    {
        Rows seq;
        auto scan = [&](int base, int64_t& w, int64_t& sum) {  // blocks of the sequences up to this thread's, and of all
            const int b = base + tid;
            if (b < a.batch) seq = rows_of(a, b);
            w = b < a.batch ? (seq.rows + kBlkRows - 1) / kBlkRows : 0;
            int64_t v = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            __syncthreads();
            if (lane == 31) ms->scan[warp] = v;
            __syncthreads();
            sum = 0;
            for (int i = 0; i < kThreads / 32; ++i) {
                if (i < warp) v += ms->scan[i];
                sum += ms->scan[i];
            }
            return v;
        };
        int64_t total = 0, w = 0, sum = 0, incl = 0;
        for (int base = 0; base < a.batch; base += kThreads) {
            incl = scan(base, w, sum);
            total += sum;
        }
        if (unit >= total) return;  // the grid is sized by a bound
        unit = (int)(total - 1 - unit);
        int64_t before = total - sum;
        for (int base = (a.batch - 1) / kThreads * kThreads;; base -= kThreads) {  // the last step's sums are at hand
            incl += before;
            if (unit >= incl - w && unit < incl) {
                ms->found[0] = base + tid;
                ms->found[1] = unit - (incl - w);
                ms->seq = seq;
            }
            if (base == 0 || unit >= before) break;
            incl = scan(base - kThreads, w, sum);
            before -= sum;
        }
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ms->kfull[i], 32 * kConvWarps);
            mbar_init(&ms->vfull[i], 32 * kConvWarps);
            mbar_init(&ms->kfree[i], PAIR ? 4 : 2);
            mbar_init(&ms->vfree[i], PAIR ? 4 : 2);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&ms->sfull[i], 1);
            mbar_init(&ms->pvd[i], 1);
            mbar_init(&ms->mpost[i], kRows);
            mbar_init(&ms->drain[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&ms->scfull[i], 32 * kConvWarps);
        mbar_init(&ms->qfull, 32 * kSoftWarps);
        ms->abort = 0;
        fence_mbar_init();
    }
    if (warp == kSoftWarps) {
        tmem_alloc(&ms->tmem, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_launch();  // not before: the next grid may take tensor memory first and then wait for this one, which waits for that memory
    const uint32_t tmem = __shfl_sync(0xffffffffu, ms->tmem, 0);
    const int b = (int)ms->found[0], row0 = (int)ms->found[1] * kBlkRows;
    const Rows sq = ms->seq;
    const int rows = min(kBlkRows, sq.rows - row0);
    // keys that the last row sees
    const int most = a.causal ? min(sq.len, max(0, sq.len - sq.n + a.by_group(row0 + rows - 1) + 1)) : sq.len;
    const int all_tiles = (most + kKeys - 1) / kKeys;
    const int t0 = (unsigned)(all_tiles * split) / (unsigned)splits, nt = (unsigned)(all_tiles * (split + 1)) / (unsigned)splits - t0;

    // The power of two that the block's query rows share: the largest finite element goes to [2^14, 2^15).
    auto common_up = [&]() {
        float big = ms->big[0];
#pragma unroll
        for (int i = 1; i < kSoftWarps; ++i) big = fmaxf(big, ms->big[i]);
        return min(253, 268 - (__float_as_int(big) >> 23));
    };

    // A row further below it than 2^6 has its own, and its scores are brought level where they are read, off the fast path. The
    // others keep the block's: fp16 parts end at 2^-24 and round at 2^-25, which is 2^-33 of such a row's largest element.
    auto up_of_row = [&](int common, int row) {
        const uint32_t bits = ms->row_big[row];
        const int own = min(253, 268 - (int)(bits >> 23));
        return bits == 0 || own - common <= 6 ? common : own;
    };

    if (warp >= kSoftWarps) {
        // ================================================================ codes to fp16 tiles
        // A warp has 32 keys of each tile. Four lanes take 64 codes of a key (one swizzled row of 128 bytes), eight keys at a
        // time; chunk i is keys 8 (i / kBlk) + lane / 4 of block i % kBlk. Stores are free of bank conflicts.
        constexpr int kBlk = HDP / 64, kChunks = 4 * kBlk;
        float rf = 0.0f;  // takes scores back to log2 units
        const int cw = warp - kSoftWarps, cc = lane & 3, rsub = lane >> 2;
        const int mask = (1 << a.c.page_shift) - 1;
        const int32_t* pg = a.pages + (int64_t)b * a.ld_pages;
        // a warp's 32 keys of a tile lie in at most two pages: those of its first and its 17th key
        int pa = 0, pb = 0;
        auto fetch = [&](int j) {
            const int k0 = (t0 + j) * kKeys + cw * 32;
            pa = k0 < sq.len ? pg[k0 >> a.c.page_shift] : 0;
            pb = k0 + 16 < sq.len ? pg[(k0 + 16) >> a.c.page_shift] : 0;
        };
        struct Where {  // this lane's chunk in its first row of the first 16 keys, and of the others less 16 rows; keys there
            int64_t ra, rb;
            uint32_t bits;
        };
        auto place = [&](int j) {
            const int k0 = (t0 + j) * kKeys + cw * 32;
            const bool ok_a = pa >= 0 && pa < a.c.n_pages, ok_b = pb >= 0 && pb < a.c.n_pages;
            if (!(ok_a && ok_b) && lane == 0) atomicOr(&g_device_error, kErrIndex);
            Where w;
            w.ra = (((int64_t)pa * a.c.kv_heads + h) << a.c.page_shift) + (k0 & mask);
            w.rb = (((int64_t)pb * a.c.kv_heads + h) << a.c.page_shift) + ((k0 + 16) & mask) - 16;
            const int left = sq.len - k0;
            w.bits = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
            if (!ok_a) w.bits &= 0xffff0000u;
            if (!ok_b) w.bits &= 0x0000ffffu;
            return w;
        };
        // The next key tile's codes wait in registers, the next value tile's in shared memory, where a thread copies the
        // chunks that it unpacks itself.
        uint4 kr[kChunks];
        uint8_t* mine = raw + (tid - 32 * kSoftWarps) * 16;
        auto load_values = [&](const Where& w) {
            const uint8_t* p[2] = {a.c.v + (w.ra + rsub) * a.c.hd + cc * 16, a.c.v + (w.rb + rsub) * a.c.hd + cc * 16};
            const uint32_t bits = w.bits >> rsub;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int k = 8 * (i / kBlk);
                const bool on = ((bits >> k) & 1) && (i % kBlk) * 64 + cc * 16 < a.c.hd;
                cp_async16(smem_u32(mine) + i * (32 * kConvWarps * 16), on ? p[k / 16] + k * a.c.hd + (i % kBlk) * 64 : a.c.v, on);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto load = [&](const uint8_t* base, const Where& w, uint4 (&r)[kChunks]) {
            const uint8_t* p[2] = {base + (w.ra + rsub) * a.c.hd + cc * 16, base + (w.rb + rsub) * a.c.hd + cc * 16};
            const uint32_t bits = w.bits >> rsub;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int k = 8 * (i / kBlk);
                r[i] = make_uint4(0, 0, 0, 0);
                if (((bits >> k) & 1) && (i % kBlk) * 64 + cc * 16 < a.c.hd)
                    r[i] = __ldg(reinterpret_cast<const uint4*>(p[k / 16] + k * a.c.hd + (i % kBlk) * 64));
            }
        };
        float ksc = 0.0f, vsc = 0.0f;
        auto load_scales = [&](const Where& w) {
            ksc = vsc = 0.0f;
            if ((w.bits >> lane) & 1) {
                const int64_t row = (lane < 16 ? w.ra : w.rb) + lane;
                ksc = __ldg(a.c.ks + row);
                vsc = __ldg(a.c.vs + row);
            }
        };
        const uint32_t at = (cw * 32 + rsub) * 128 + (((2 * cc) ^ rsub) << 4), k_at = smem_u32(sK) + at, v_at = smem_u32(sV) + at;
        auto store = [&](uint32_t tile, int i, uint4 r) {
            uint32_t w[8];
            unpack4<E4M3>(r.x, w[0], w[1]);
            unpack4<E4M3>(r.y, w[2], w[3]);
            unpack4<E4M3>(r.z, w[4], w[5]);
            unpack4<E4M3>(r.w, w[6], w[7]);
            const int off = (i % kBlk) * kBlock + (i / kBlk) * 1024;
            st_shared16(tile + off, make_uint4(w[0], w[1], w[2], w[3]));
            st_shared16((tile ^ 16) + off, make_uint4(w[4], w[5], w[6], w[7]));
        };
        // Order of the tiles: K0, K1, V0, K2, V1, ...: the next tile's scores do not wait for this one's V. Each is asked for
        // when the one before it of its kind has been stored.
        Where pk{}, pv{};  // places of the keys and values asked for last
        auto ask_keys = [&](int j) {
            pv = pk;
            if (j >= nt) return;
            pk = place(j);
            load(a.c.k, pk, kr);
            load_scales(pk);
            if (j + 1 < nt) fetch(j + 1);
        };
        auto keys = [&](int j) {
            const int st = j & 1, sc = j & 3;
            if (j >= 2) wait(ms, &ms->kfree[st], (uint32_t)((j >> 1) - 1) & 1u);
#pragma unroll
            for (int i = 0; i < kChunks; ++i) store(k_at + st * kTileBytes, i, kr[i]);
            fence_proxy_async_smem();
            mbar_arrive(&ms->kfull[st]);
            if (j == 0) {
                wait(ms, &ms->qfull, 0);
                rf = __fmul_rn(pow2_biased(254 - common_up()), a.scale_log2e);
            }
            const float kf = __fmul_rn(ksc, rf);
            ms->ks[sc][cw * 32 + lane] = kf;
            ms->vs[sc][cw * 32 + lane] = vsc;
            int e = __float_as_int(fabsf(vsc)) >> 23;
            e = __reduce_max_sync(0xffffffffu, e == 255 ? 1 : max(1, min(252, e)));
            ms->vn[sc][cw * 32 + lane] = __fmul_rn(vsc, pow2_biased(253 - e));
            // elements of Q are below 2^15, codes below 2^9 and 2^7
            const bool wide = __any_sync(0xffffffffu, !(fabsf(kf) < 0x1p9f / (HDP * (E4M3 ? 512 : 128))));
            if (lane == 0) {
                ms->of[sc][cw >> 1].vexp[cw & 1] = wide ? e | kWide : e;
                ms->of[sc][cw >> 1].there[cw & 1] = pk.bits;
            }
            __syncwarp();
            mbar_arrive(&ms->scfull[sc]);
        };
        if (nt > 0) fetch(0);
#pragma unroll 1
        for (int j = -2; j < nt; ++j) {  // one copy of each step: the code of a turn has to stay in the instruction cache
            const bool more = j >= -1 && j + 1 < nt;
            if (more) keys(j + 1);
            ask_keys(j + 2);
            if (j >= 0) {
                if (j >= 2) wait(ms, &ms->vfree[j & 1], (uint32_t)((j >> 1) - 1) & 1u);
                asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
                for (int i = 0; i < kChunks; ++i)
                    store(v_at + (j & 1) * kTileBytes, i, *reinterpret_cast<const uint4*>(mine + i * (32 * kConvWarps * 16)));
                fence_proxy_async_smem();
                mbar_arrive(&ms->vfull[j & 1]);
            }
            if (more) load_values(pv);
        }
    } else {
        // ================================================================ softmax
        int common;
        // ---- the query rows, 16 bytes a lane: two bf16 rows or one fp32 row for each warp and load
        {
            constexpr int kPer = PARTS == 2 ? 1 : 2, kQr = kBlkRows / kSoftWarps / kPer;
            constexpr int kVals = PARTS == 2 ? 4 : 8, kLanes = 32 / kPer;
            const int sub = lane / kLanes, d = (lane % kLanes) * kVals, dd = min(d, a.c.hd - kVals);
            uint4 q[kQr];
            const int first = warp * kPer + sub;  // rows first, first + 16 kPer, ...
#pragma unroll
            for (int k = 0; k < kQr; ++k) {  // all loads are in flight before the first is used; what is not there is dropped
                const int rr = row0 + min(first + k * kSoftWarps * kPer, rows - 1), ti = a.by_group(rr);
                const int64_t at = (sq.lo + (int64_t)ti) * a.ldq + (int64_t)(h * a.group + (rr - ti * a.group)) * a.c.hd + dd;
                q[k] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) + at * (PARTS == 2 ? 4 : 2));
            }
            auto values = [&](uint4 u, bool on, float (&x)[kVals]) {
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < kVals; ++i) {
                    const float y = PARTS == 2 ? __uint_as_float(w[i & 3])
                                               : __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
                    x[i] = on ? y : 0.0f;
                }
            };
            uint32_t big = 0;
#pragma unroll
            for (int k = 0; k < kQr; ++k) {
                float x[kVals];
                values(q[k], first + k * kSoftWarps * kPer < rows && d < a.c.hd, x);
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < kVals; ++i) bits = max(bits, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
                if (d == 0) ms->row_big[first + k * kSoftWarps * kPer] = bits;
                big = max(big, bits < 0x7f800000u ? bits : 0u);
            }
            big = __reduce_max_sync(0xffffffffu, big);
            if (lane == 0) ms->big[warp] = __uint_as_float(big);
            asm volatile("bar.sync 1, 512;" ::: "memory");
            common = common_up();
            if (d < HDP) {
#pragma unroll
                for (int k = 0; k < kQr; ++k) {
                    const int r = first + k * kSoftWarps * kPer, rr = r & (kRows - 1);
                    float x[kVals];
                    values(q[k], r < rows && d < a.c.hd, x);
                    const float mul = pow2_biased(up_of_row(common, r));
                    uint32_t hi[kVals / 2];
                    float y[kVals];
#pragma unroll
                    for (int i = 0; i < kVals; i += 4) {  // in the order of unpack4's pairs
                        y[i] = __fmul_rn(x[i], mul);
                        y[i + 1] = __fmul_rn(x[i + (E4M3 ? 1 : 2)], mul);
                        y[i + 2] = __fmul_rn(x[i + (E4M3 ? 2 : 1)], mul);
                        y[i + 3] = __fmul_rn(x[i + 3], mul);
                        hi[i / 2] = pack_h2(y[i], y[i + 1]);
                        hi[i / 2 + 1] = pack_h2(y[i + 2], y[i + 3]);
                    }
                    uint8_t* p = sQ + (PAIR ? (r >> 7) * kTileBytes : 0) + (d >> 6) * kBlock + rr * 128 +
                                 ((((d & 63) >> 3) ^ (rr & 7)) << 4) + (d & 4) * 2;
                    if constexpr (PARTS == 1) {
                        *reinterpret_cast<uint4*>(p) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    } else {
                        *reinterpret_cast<uint2*>(p) = make_uint2(hi[0], hi[1]);
                        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&hi[0]));
                        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi[1]));
                        *reinterpret_cast<uint2*>(p + kTileBytes) =
                            make_uint2(pack_h2(__fsub_rn(y[0], f0.x), __fsub_rn(y[1], f0.y)),
                                       pack_h2(__fsub_rn(y[2], f1.x), __fsub_rn(y[3], f1.y)));
                    }
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&ms->qfull);
        }
        const int wg = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
        const int st = 2 * wg + half;  // stream
        const uint32_t sbuf = lane_addr + st * kHalf, obuf = lane_addr + kOcol + wg * kRows;
        const int rb = row0 + (PAIR ? wg * kRows : 0) + r;  // row of the sequence
        const bool mine = rb < row0 + rows;
        const int tok = a.by_group(rb);
        // a row that is not there never masks (its results are dropped)
        const int limit = !mine ? 0x7fffffff : a.causal ? sq.len - sq.n + tok + 1 : sq.len;
        const int n = PAIR ? nt : (nt + 1 - wg) / 2;
        // 0, or the power of two that takes the row's scores level; 1: an infinity or a NaN makes them NaN
        auto drop = [&](int up) {
            const int row = (PAIR ? wg * kRows : 0) + r;
            return ms->row_big[row] >= 0x7f800000u ? 1 : up - up_of_row(up, row);
        };
        const int wmin = __reduce_min_sync(0xffffffffu, drop(common) == 0 ? limit : -1);  // keys that all of the warp's rows see as they are
        auto level = [&](auto& x) {
            if (wmin >= 0) return;
            const int by = drop(common_up());
            const float f0 = by > 0 ? __int_as_float(0x7fc00000) : pow2_biased(127 + max(by, -120)), f1 = pow2_biased(127 + max(min(by + 120, 0), -126));
            for (auto& v : x) v = __float_as_uint(__fmul_rn(__fmul_rn(__uint_as_float(v), f0), f1));
        };
        float m = -INFINITY, l = 0.0f;  // reference and sum of this thread's keys
        int vref = 12;
        // ---- this stream's MMAs, issued by one of its warps: another scheduler's for each stream
        const bool leader = quad == st;
        const uint32_t q0 = smem_u32(sQ) + (PAIR ? wg * kTileBytes : 0), s0 = tmem + st * kHalf, o0 = tmem + kOcol + wg * kRows;
        volatile int* ab = &ms->abort;
        auto issue_scores = [&](int i) {
            const int j = PAIR ? i : 2 * i + wg;
            wait(ms, &ms->kfull[j & 1], (uint32_t)(j >> 1) & 1u);
            if (__any_sync(0xffffffffu, *ab)) return;
            tc_fence_after();
            const uint32_t kt = smem_u32(sK) + (j & 1) * kTileBytes + half * (kHalf * 128);
            const uint64_t qd = umma_desc_k_sw128(q0), kd = umma_desc_k_sw128(kt);
#pragma unroll
            for (int k = 0; k < PARTS * (HDP / 16); ++k) {  // the small part first: fewer roundings of large sums
                const int part = PARTS - 1 - k / (HDP / 16), s = k % (HDP / 16);
                const uint32_t off = ((s >> 2) * kBlock + (s & 3) * 32) >> 4;
                mma_ss(s0, qd + (part * kTileBytes >> 4) + off, kd + off, idesc_f16(kHalf, false), k > 0 ? 1u : 0u);
            }
            commit_elected(&ms->sfull[st]);
            commit_elected(&ms->kfree[j & 1]);
        };
        auto issue_outputs = [&](int i) {
            const int j = PAIR ? i : 2 * i + wg;
            wait(ms, &ms->vfull[j & 1], (uint32_t)(j >> 1) & 1u);
            // behind the other stream's product, so that the order of the sums is always the same
            if (i + half > 0) wait(ms, &ms->pvd[st ^ 1], (uint32_t)(half ? i : i - 1) & 1u);
            if (__any_sync(0xffffffffu, *ab)) return;
            tc_fence_after();
            const uint32_t vt = smem_u32(sV) + (j & 1) * kTileBytes + half * (kHalf * 128);
            const uint64_t vd = desc_mn_sw128(vt);
#pragma unroll
            for (int k = 0; k < 2 * (kHalf / 16); ++k) {  // P of 32 keys: 16 columns of the large parts, 16 of the small ones
                const int part = 1 - k / (kHalf / 16), s = k % (kHalf / 16);
                mma_ts(o0, s0 + (s >> 1) * 32 + part * 16 + (s & 1) * 8, vd + (s * 2048 >> 4), idesc_f16(HDP, true),
                       k > 0 ? 1u : i + half > 0 ? 1u : 0u);
            }
            commit_elected(&ms->pvd[st]);
            commit_elected(&ms->vfree[j & 1]);
        };
        if (leader) wait(ms, &ms->qfull, 0);
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int j = PAIR ? i : 2 * i + wg, sc = j & 3;
            if (leader) {
                if (i > 0) wait(ms, &ms->pvd[st], (uint32_t)(i - 1) & 1u);  // these scores overwrite P
                issue_scores(i);
            }
            __syncwarp();
            wait(ms, &ms->scfull[sc], (uint32_t)(j >> 2) & 1u);
            const int4 of = *reinterpret_cast<const int4*>(&ms->of[sc][half]);
            const int key0 = (t0 + j) * kKeys + half * kHalf;
            // not plain: keys that a row does not see, rows to be brought level, or scores for which a product that is not rounded
            // may differ from its reference by more than a half
            const bool plain = !__any_sync(0xffffffffu, (of.x & of.y) != -1 || key0 + kHalf > wmin || ((of.z | of.w) & kWide));
            // keys of 32 that the row sees
            auto see_of = [&](int c) {
                const int left = limit - (key0 + 32 * c);
                return ms->of[sc][half].there[c] & (left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u);
            };
            wait(ms, &ms->sfull[st], (uint32_t)i & 1u);
            tc_fence_after();
            // 2^(from - to) for whole numbers from <= to; 0 from -inf
            auto down = [&](float from, float to) {
                const float by = __fsub_rn(from, to);
                return by >= -126.0f ? pow2_biased(127 + (int)by) : 0.0f;
            };
            auto part = [&](F2 w, uint32_t& hi, uint32_t& lo) {
                float u, v;
                unf2(w, u, v);
                hi = pack_h2(u, v);
                const float2 b2 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                unf2(add2(w, f2(-b2.x, -b2.y)), u, v);
                lo = pack_h2(u, v);
            };
            // The half tile's first chunks of 32 keys. The parts are put together, multiplied and split anew: an fp16 factor ends at
            // 2^-24, where a jump of the scores or of the value scales does not, and parts scaled by themselves lose their low bits.
            auto scale_probabilities = [&](int chunks, float f) {
                tc_wait_st();
#pragma unroll 1
                for (int c = 0; c < 2 * chunks; ++c) {
                    const uint32_t at = sbuf + 32 * (c >> 1) + 8 * (c & 1);
                    uint32_t hi[8], lo[8];
                    tmem_ld_x8(at, hi);
                    tmem_ld_x8(at + 16, lo);
                    wait_ld(hi, lo);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
                        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&lo[k]));
                        part(mul2(add2(f2(h.x, h.y), f2(g.x, g.y)), f2(f, f)), hi[k], lo[k]);
                    }
                    tmem_st_x8(at, hi);
                    tmem_st_x8(at + 16, lo);
                }
            };
            if (plain) {
                const int e = max(of.z, of.w);
                if (e >= vref) vref = min(e + 2, 255);
                // P of 32 keys over their scores: p = 2^(s - m + shift) times the value scales, which are over 2^(exponent + 1)
                // of their 32 keys (one far below the reference counts as 2^-60); their sum is taken back by 2^-shift. With
                // shift = 9, or 10 where the exponent has grown by one, P stays below 2^15, and its small parts, which end at
                // 2^-24, round the row's largest product of probability and value scale at 2^-33 of it (2^-32 where its score
                // is a unit below the reference)
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    const float4* ksp = reinterpret_cast<const float4*>(&ms->ks[sc][half * kHalf + 32 * c]);
                    const float4* vnp = reinterpret_cast<const float4*>(&ms->vn[sc][half * kHalf + 32 * c]);
                    const int shift = max(-60, ms->of[sc][half].vexp[c] + 11 - vref);
                    const float most = pow2_biased(127 + 5 + shift);
                    uint32_t x[32];
                    float sum;
                    tmem_ld_32x32b_x32(sbuf + 32 * c, x);
                    wait_ld(x);
                    for (bool again = false;; again = true) {
                        const float cc = __fsub_rn((float)shift, m);
                        const F2 c2 = f2(cc, cc);
                        F2 sum0 = f2(0.0f, 0.0f), sum1 = sum0;
                        float u, v;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {  // P of 16 keys at a time
                            uint32_t hi[8], lo[8];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float4 f = ksp[4 * q + k], g = vnp[4 * q + k];
                                const uint32_t* xk = &x[16 * q + 4 * k];
                                unf2(fma2(f2u(xk[0], xk[1]), f2(f.x, f.y), c2), u, v);
                                F2 p = f2(ex2(u), ex2(v));
                                sum0 = add2(sum0, p);
                                part(mul2(p, f2(g.x, g.y)), hi[2 * k], lo[2 * k]);
                                unf2(fma2(f2u(xk[2], xk[3]), f2(f.z, f.w), c2), u, v);
                                p = f2(ex2(u), ex2(v));
                                sum1 = add2(sum1, p);
                                part(mul2(p, f2(g.z, g.w)), hi[2 * k + 1], lo[2 * k + 1]);
                            }
                            tmem_st_x8(sbuf + 32 * c + 8 * q, hi);
                            tmem_st_x8(sbuf + 32 * c + 16 + 8 * q, lo);
                        }
                        unf2(add2(sum0, sum1), u, v);
                        sum = __fadd_rn(u, v);
                        // too large at first (m is -inf), where the scores have grown, and for NaN
                        if (again || !__any_sync(0xffffffffu, !(sum <= most))) break;
                        float mx = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float4 f = ksp[k];
                            mx = max3(mx, __fmul_rn(__uint_as_float(x[4 * k]), f.x), __fmul_rn(__uint_as_float(x[4 * k + 1]), f.y));
                            mx = max3(mx, __fmul_rn(__uint_as_float(x[4 * k + 2]), f.z), __fmul_rn(__uint_as_float(x[4 * k + 3]), f.w));
                        }
                        float f = 1.0f;
                        if (mx > m) {
                            const float mn = ceilf(mx);
                            f = down(m, mn);
                            l = __fmul_rn(l, f);
                            m = mn;
                        }
                        if (c > 0) scale_probabilities(1, f);
                    }
                    l = __fmaf_rn(sum, pow2_biased(127 - shift), l);
                }
            } else {  // a key or value scale that the row does not see may be anything
                float mx = -INFINITY, vmx = 0.0f;
                const float* kp = &ms->ks[sc][half * kHalf];
                const float* vp = &ms->vs[sc][half * kHalf];
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const uint32_t see = (see_of(c >> 1) >> (16 * (c & 1))) & 0xffffu;
                    if (!__any_sync(0xffffffffu, see)) continue;  // mostly so on a causal diagonal: 32 rows are few tokens
                    uint32_t x[16];
                    tmem_ld_x16(sbuf + 16 * c, x);
                    wait_ld(x);
                    level(x);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float u = __fmul_rn(__uint_as_float(x[k]), kp[16 * c + k]);
                        if ((see >> k) & 1) {
                            mx = fmaxf(mx, u);
                            vmx = fmaxf(vmx, fabsf(vp[16 * c + k]));
                        }
                    }
                }
                const int e = __float_as_int(vmx) >> 23;
                if (e >= vref) vref = min(e + 2, 255);
                if (mx > __fadd_rn(m, 5.0f)) {
                    const float mn = ceilf(mx);
                    l = __fmul_rn(l, down(m, mn));
                    m = mn;
                }
                const float mu = m == -INFINITY ? 0.0f : -m, vmul = pow2_biased(264 - vref);
                uint32_t keep[8];
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const uint32_t see = (see_of(c >> 1) >> (16 * (c & 1))) & 0xffffu;
                    float sum = 0.0f;
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) hi[k] = lo[k] = 0;
                    if (__any_sync(0xffffffffu, see)) {
                        uint32_t x[16];
                        tmem_ld_x16(sbuf + 16 * c, x);
                        wait_ld(x);
                        level(x);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float p[2], w[2];
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const int key = 16 * c + 2 * k + q;
                                const bool on = (see >> (2 * k + q)) & 1;
                                p[q] = on ? ex2(__fadd_rn(__fmul_rn(__uint_as_float(x[2 * k + q]), kp[key]), mu)) : 0.0f;
                                w[q] = on ? __fmul_rn(p[q], __fmul_rn(vp[key], vmul)) : 0.0f;
                            }
                            sum = __fadd_rn(sum, __fadd_rn(p[0], p[1]));
                            part(f2(w[0], w[1]), hi[k], lo[k]);
                        }
                    }
                    const uint32_t to = sbuf + 32 * (c >> 1) + 8 * (c & 1);
                    // the chunk's second 16 scores lie where its small parts go: they are kept until those are read
                    if (c & 1) {
                        tmem_st_x8(to, hi);
                        tmem_st_x8(to + 16, lo);
                        tmem_st_x8(to + 8, keep);
                    } else {
                        tmem_st_x8(to, hi);
#pragma unroll
                        for (int k = 0; k < 8; ++k) keep[k] = lo[k];
                    }
                    l = __fadd_rn(l, sum);
                }
            }
            // ---- one reference for the row's outputs: the other stream has left the one that its last half tile went in with
            if (i + half > 0) wait(ms, &ms->mpost[st ^ 1], (uint32_t)(half ? i : i - 1) & 1u);
            const float mo = i + half > 0 ? ms->om[wg][r] : -INFINITY;
            const int vo = i + half > 0 ? ms->ov[wg][r] : 12;
            if (__any_sync(0xffffffffu, m != mo || vref != vo)) {
                const float mn = fmaxf(m, mo);
                const int vn = max(vref, vo);
                const float fm = m == mn ? 1.0f : down(m, mn);
                const float fp = __fmul_rn(fm, vn - vref > 126 ? 0.0f : pow2_biased(127 - (vn - vref)));
                const float fo = __fmul_rn(mo == mn ? 1.0f : down(mo, mn), vn - vo > 126 ? 0.0f : pow2_biased(127 - (vn - vo)));
                l = __fmul_rn(l, fm);
                if (__any_sync(0xffffffffu, fp != 1.0f)) scale_probabilities(2, fp);
                if (i + half > 0 && __any_sync(0xffffffffu, fo != 1.0f)) {
                    wait(ms, &ms->pvd[st ^ 1], (uint32_t)(half ? i : i - 1) & 1u);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HDP; c += 16) {
                        uint32_t x[16];
                        tmem_ld_x16(obuf + c, x);
                        wait_ld(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(__fmul_rn(__uint_as_float(x[k]), fo));
                        tmem_st_x16(obuf + c, x);
                    }
                }
                m = mn;
                vref = vn;
            }
            ms->om[wg][r] = m;
            ms->ov[wg][r] = vref;
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&ms->mpost[st]);
            asm volatile("bar.sync %0, 128;" ::"r"(2 + st) : "memory");
            tc_fence_after();
            if (leader) issue_outputs(i);
            __syncwarp();
        }
        if (n > 0) {  // the second stream's last product is the group's last
            wait(ms, &ms->pvd[st | 1], (uint32_t)(n - 1) & 1u);
            tc_fence_after();
        }
        if (leader) {  // also after a wait that ran out: what was issued finishes before tensor memory is freed
            commit_elected(&ms->drain[st]);
            mbar_wait(&ms->drain[st], 0, 2u);
        }
        __syncwarp();
        // ---- results: half of the columns of its row for each thread, a quarter where both groups have the same rows
        if (n == 0) {
            ms->om[wg][r] = -INFINITY;
            ms->ov[wg][r] = 12;
        } else {
            wait(ms, &ms->mpost[st | 1], (uint32_t)(n - 1) & 1u);
            const float mf = ms->om[wg][r];  // the last reference
            if (m != mf) l = m == -INFINITY ? 0.0f : __fmul_rn(l, ex2(__fsub_rn(m, mf)));
        }
        ms->l[wg][half][r] = l;
        tc_fence_before();
        asm volatile("bar.sync 1, 512;" ::: "memory");  // every product has been made: Q and K are not read any more
        tc_fence_after();
        float f0 = pow2_biased(ms->ov[wg][r] - 10), f1 = 0.0f;
        m = ms->om[wg][r];
        l = __fadd_rn(ms->l[wg][0][r], ms->l[wg][1][r]);
        if (!PAIR) {
            const float ma = ms->om[0][r], mb = ms->om[1][r];
            m = fmaxf(ma, mb);
            const float fa = ma == -INFINITY ? 0.0f : ex2(__fsub_rn(ma, m)), fb = mb == -INFINITY ? 0.0f : ex2(__fsub_rn(mb, m));
            l = __fmaf_rn(__fadd_rn(ms->l[0][0][r], ms->l[0][1][r]), fa, __fmul_rn(__fadd_rn(ms->l[1][0][r], ms->l[1][1][r]), fb));
            f0 = __fmul_rn(pow2_biased(ms->ov[0][r] - 10), fa);
            f1 = __fmul_rn(pow2_biased(ms->ov[1][r] - 10), fb);
        }
        const int c0 = PAIR ? half * (HDP / 2) : (2 * wg + half) * (HDP / 4), c1 = c0 + (PAIR ? HDP / 2 : HDP / 4);
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        if (a.to_state && mine && c0 == 0) {
            const int64_t si = ((int64_t)split * a.M + sq.lo + tok) * a.heads + h * a.group + (rb - tok * a.group);
            a.out.m[si] = m;
            a.out.l[si] = l;
        }
        // Rows go through shared memory, over Q (fp32 pieces of bf16 rows also over K), so that a warp writes whole ones
        const int lg = PARTS == 2 || a.to_state ? 2 : 1;  // bytes of an element, as a shift
        uint8_t* to = sQ + (((PAIR ? wg * kRows : 0) + r) * HDP << lg);
        const uint32_t oa = lane_addr + kOcol + (PAIR ? wg * kRows : 0);
#pragma unroll 1
        for (int d = c0; d < c1; d += 16) {
            uint32_t x[16], y[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = y[k] = 0;
            if (nt > 0) tmem_ld_x16(oa + d, x);
            if (!PAIR && nt > 1) tmem_ld_x16(oa + kRows + d, y);
            wait_ld(x);
            if (!PAIR) wait_ld(y);
            if (d >= a.c.hd) continue;
            float o[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                o[k] = __fmul_rn(__uint_as_float(x[k]), f0);
                if (!PAIR) o[k] = __fmaf_rn(__uint_as_float(y[k]), f1, o[k]);
            }
            if (!E4M3) {  // out of the order of unpack4's pairs
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float z = o[k + 1];
                    o[k + 1] = o[k + 2];
                    o[k + 2] = z;
                }
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = a.to_state ? o[k] : l == 0.0f ? 0.0f : __fmul_rn(o[k], inv);
            if (lg == 1) {
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const __nv_bfloat162 z = __floats2bfloat162_rn(o[2 * k], o[2 * k + 1]);
                    w[k] = *reinterpret_cast<const uint32_t*>(&z);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    *reinterpret_cast<uint4*>(to + (((d >> 3) + k) ^ (r & 7)) * 16) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<float4*>(to + (((d >> 2) + k) ^ (r & 7)) * 16) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
        }
        asm volatile("bar.sync 1, 512;" ::: "memory");
        const int sh = (HDP == 128 ? 3 : 2) + lg, per = 1 << sh;  // 16-byte pieces of a row
#pragma unroll 4
        for (int i = tid; i < rows * per; i += 32 * kSoftWarps) {
            const int rr = i >> sh, c = i & (per - 1), t = a.by_group(row0 + rr);
            const uint4 u = *reinterpret_cast<const uint4*>(sQ + (rr * HDP << lg) + (c ^ (rr & 7)) * 16);
            if (c << (4 - lg) >= a.c.hd) continue;
            const int64_t grow = sq.lo + (int64_t)t;
            const int head = h * a.group + (row0 + rr - t * a.group);
            uint8_t* p = a.to_state ? reinterpret_cast<uint8_t*>(a.out.o + (((int64_t)split * a.M + grow) * a.heads + head) * a.c.hd)
                                    : static_cast<uint8_t*>(a.o) + ((grow * a.ldo + (int64_t)head * a.c.hd) << lg);
            *reinterpret_cast<uint4*>(p + c * 16) = u;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSoftWarps) {
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
        auto has = [&](int b) {
            const int first = a.q_start[b], end = a.q_start[b + 1];
            return first >= 0 && first <= row && row < end && end <= a.M;
        };
        if (lo < 0 || !has(lo)) {
            // behind the last sequence, or an entry out of order has led the search astray
            if (lo == a.batch - 1 && a.q_start[lo] >= 0) continue;
            int found = a.batch;
            for (int b = lane; b < a.batch && found == a.batch; b += 32)
                if (has(b)) found = b;
            lo = __reduce_min_sync(0xffffffffu, found);
            if (lo == a.batch) continue;
        }
        const Rows sq = rows_of(a, lo);
        if (sq.rows == 0) continue;
        if (a.add.pieces > 0 && sq.lo + sq.n > rows_used(a, a.q_start[a.batch])) continue;  // no state from the prefix
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

template <int HDP, bool E4M3, int PARTS, bool PAIR>
cudaError_t launch_typed(const KvAttnArgs& a, int splits, cudaStream_t st) {
    auto kernel = kv_attention_tc_kernel<HDP, E4M3, PARTS, PAIR>;
    const size_t smem = kSmem<HDP, PARTS, PAIR>;
    const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    // blocks of rows at most: one more than whole ones for each sequence that has rows enough
    const int64_t units = a.M * a.group / (PAIR ? 2 * kRows : kRows) + std::min<int64_t>(a.batch, a.M * a.group / (a.min_rows + 1));
    if (units == 0) return cudaSuccess;
    return launch_pdl(kernel, units * a.c.kv_heads * splits, kThreads, smem, st, a, (int)units, splits);
}
template <int HDP, bool E4M3>
cudaError_t launch_code(const KvAttnArgs& a, bool pair, int splits, cudaStream_t st) {
    if (!a.bf16) return launch_typed<HDP, E4M3, 2, false>(a, splits, st);
    return pair ? launch_typed<HDP, E4M3, 1, true>(a, splits, st) : launch_typed<HDP, E4M3, 1, false>(a, splits, st);
}

}  // namespace

cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, bool pair, int splits, cudaStream_t st) {
    if (a.batch <= 0 || a.M <= 0) return cudaSuccess;
    if (a.c.hd > 64) return a.c.e4m3 ? launch_code<128, true>(a, pair, splits, st) : launch_code<128, false>(a, pair, splits, st);
    return a.c.e4m3 ? launch_code<64, true>(a, pair, splits, st) : launch_code<64, false>(a, pair, splits, st);
}

cudaError_t launch_kv_state_join(const KvAttnArgs& a, cudaStream_t st) {
    const int64_t blocks = ceil_div(a.M * a.heads, kJoinThreads / 32);
    return launch_pdl(kv_state_join_kernel, blocks < 148 * 8 ? blocks : 148 * 8, kJoinThreads, 0, st, a);
}

}  // namespace b2s
