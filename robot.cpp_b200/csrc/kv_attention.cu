// kv_attention.cu -- attention of few query rows for each key/value head over the paged 8-bit cache: decoding steps,
// drafts and short tails. One pass over the keys with the running maximum and sum of the softmax.
//
// Floor: the cache bytes, (2 hd + 8) per token and key/value head. A decoding step does 4 * group * hd operations on
// them, so the products only have to keep up with memory.
//
//   score(j) = q . code(j) * k_scale(j) * scale * log2 e;   p(j) = 2^(score - m);
//   o = sum p(j) v_scale(j) code(j) / sum p(j)
// Products: warp-level MMAs with fp32 or int32 accumulation. 8-bit codes (int8 and e4m3) are exact in fp16, so only the
// fp32 side of a product is split. The eight rows of a unit are MMA rows 0-7 with their larger and 8-15 with their smaller
// part: one MMA gives both and their sum is in one thread.
//   e4m3 scores: a query row, scaled by the power of two that brings its largest element to 2^14, is hi + lo with hi =
//     fp16(x), lo = fp16(x - hi): relative error 2^-22, elements 2^-38 below the largest one lose bits.
//   int8 scores: the row as integers of 24 bits under its largest element (error 2^-24 of that), in three signed bytes; the
//     codes go into m16n8k32 integer MMAs as they lie in memory. Unpacking them to fp16 had cost five instructions for four
//     codes and kept the integer pipe busier than memory.
//   outputs: the probabilities times the value scale as hi + lo, codes unpacked to fp16. The value scales are brought into
//     fp16's range by a power of two above the largest one seen (vref).
//
// Split: a unit is (sequence, key/value head, eight query rows), its keys are tiles of 32. All units' tiles, laid end to
// end, are cut into equal ranges, one for each resident block, so that uneven lengths load every SM alike. A block's
// four warps take the tiles of its range in turn, each through its own ring of asynchronous copies (no block-wide
// wait between tiles, the ring runs on across units); at a unit's end they are joined through shared memory. A unit cut
// by a range's border leaves partial results that kv_attention_join_kernel puts together: the order is fixed by the
// lengths alone, so results do not change from run to run. Short units are not cut, and many short ones go to a warp each.
//
// Measured, 20 heads on 5 of 128, one fp32 row a sequence, int8: 64 sequences of 1024..8192 tokens 95 us, 4.4 TB/s of a copy's
// 6.5; 64 of 8192 tokens 132 us, 5.2 TB/s (e4m3 and bf16 125-133 us); one of 32768 29 us; one of 317 9.7-11 us. What bounds it is
// the warps' own work between two tiles (issue slots 53% busy, memory 53%), then starting and joining units.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "b2s_internal.h"
#include "kv_internal.h"

namespace b2s {

namespace kva {
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kTile = 32;   // keys per warp step
constexpr int kRows = 8;    // query rows of a unit
constexpr int kStages = 2;
constexpr int kPerSm = 3, kMaxCtas = kPerSm * 160;
constexpr int kMinTiles = 8;  // a block gets at least this many tiles (two steps of each warp); 2 or 32 cost 4 x 2000 keys 20%, 60%
// Units that cannot have more tiles are not cut: nothing is left to join. 64 x 5 units of 500 tokens 17 us against 30 cut ones, of
// 700 20 against 29; one sequence of 700 14.6 against 14.0, of 1500 24 (not cut) against 15.
constexpr int kWholeTiles = 24;
// Nor are units of at most this many tiles shared by a block's warps, if they are many: 8 units > (8 + tiles) blocks. Five heads, us
// with a unit a block and a unit a warp: 128 sequences of 30 tokens 15.3 and 10.4, 512 42 and 21; 128 of 100 17.1 and 18.2, 256
// 26 and 20, 512 51 and 38; 128 of 300 27 and 34, 256 40.4 and 38.7, 512 77 and 69; 512 of 600 111 and 114. A warp alone takes
// 1.4 us a tile, so few units or long ones are better shared.
constexpr int kSoloTiles = 12;
template <int HD>
constexpr int kStageBytes = 2 * kTile * HD + 2 * kTile * 4 + 128;  // K, V codes, scales, which keys are there
template <int HD>
constexpr int kPart = kRows * HD + 2 * kRows;  // floats of a partial result: o, m, l
// What block c says of the border in front of it, for the join: the pieces of the unit that it cuts, if it is the first one
// there, and the unit's rows.
struct Border {
    int pieces;  // of blocks c - 1, c, ...; 0: nothing to join
    int slot;    // where block c - 1 left its piece
    int lo, head0, row0, rows;
};
}  // namespace kva

namespace {

using namespace kva;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e of a biased exponent 1..254.
__device__ __forceinline__ float pow2_biased(int e) { return __int_as_float(e << 23); }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// m16n8k32 on signed bytes.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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
// hi and lo fp16 parts of two values, packed (x0 in the low half).
__device__ __forceinline__ void split_h2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(__fsub_rn(x0, f.x), __fsub_rn(x1, f.y));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Two pairs of fp16 codes from two words of bytes whose 16-bit halves are {a0 a1}, {b0 b1} in x (e4m3: {a0 b0}, {a1 b1}).
// int8: 1024 + (b + 128) is the fp16 number 0x6400 | (b ^ 0x80); 1152 is taken off again. Both steps are exact.
template <bool E4M3>
__device__ __forceinline__ void unpack4(uint32_t x, uint32_t& p0, uint32_t& p1) {
    if (E4M3) {
        p0 = e4m3x2_to_h2(x);
        p1 = e4m3x2_to_h2(x >> 16);
    } else {
        p0 = sub_h2((x & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
        p1 = sub_h2(((x >> 8) & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u);
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    const int n = on ? 16 : 0;  // 0 bytes: nothing is read, zeros are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool on) {
    const int n = on ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---------------------------------------------------------------- units
// A sequence's keys as the kernel counts them: a shared prefix padded to whole tiles, then its own.
struct Seq {
    int lo, n, len;    // first query row, query rows, keys
    int row_tiles, units, tiles;
};

__device__ __forceinline__ Seq seq_of(const KvAttnArgs& a, int b) {
    Seq s;
    const int lo = a.q_start[b * a.q_stride], hi = a.q_start[(b + 1) * a.q_stride];
    int64_t len = a.kv_len ? (int64_t)a.kv_len[b] : a.kv_const;
    const int64_t cap = a.max_pages << a.c.page_shift;
    bool bad = lo < 0 || hi < lo || hi > a.M || (a.add.pieces > 0 && hi > rows_used(a, a.q_start[a.batch]));
    s.lo = lo;
    s.n = bad ? 0 : hi - lo;
    if (len < 0 || len > cap) {
        bad = true;
        len = len < 0 ? 0 : cap;
    }
    if (bad) atomicOr(&g_device_error, kErrIndex);
    s.len = a.prefix_pad + (int)len;
    const int rows = s.n * a.group;
    s.row_tiles = rows > a.min_rows && rows <= a.max_rows ? (rows + kRows - 1) / kRows : 0;
    s.units = s.row_tiles * a.c.kv_heads;
    s.tiles = s.len > kTile ? (s.len + kTile - 1) / kTile : 1;
    return s;
}
// What ranges are cut in: tiles, or whole units.
__device__ __forceinline__ int64_t work_of(const Seq& s, const KvAttnArgs& a) {
    return a.whole_units ? (int64_t)s.units : (int64_t)s.units * s.tiles;
}

struct Place {
    int b;
    int64_t off;  // into the sequence's work
};

// Inclusive sum of v over the block's threads, and the block's total.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sh, int64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh[w];
        total += sh[w];
    }
    return v + before;
}

// Whole-number quotient; most are of numbers below 2^32, which divide several times faster.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
    return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}
// The total in equal shares: the first `more` blocks have one tile more.
struct Ranges {
    int64_t total, share;
    int ctas, more;
    __device__ __forceinline__ int64_t start(int c) const { return share * c + min(c, more); }
    // the block that tile x falls to
    __device__ __forceinline__ int owner(int64_t x) const {
        const int64_t big = (share + 1) * more;
        return x < big ? (int)quotient(x, share + 1) : more + (int)quotient(x - big, share);
    }
};

// All threads: the total of tiles, how many workers (blocks, or N = kWarps warps each) share them, and the places of the first
// tiles of the block's workers c, c + 1, ... below ctas.
template <int N>
__device__ __forceinline__ Ranges find_range(const KvAttnArgs& a, int c, int64_t* sh, Place (&sh_place)[N]) {
    int64_t total = 0, w = 0, incl = 0, sum;
    for (int base = 0; base < a.batch; base += kThreads) {
        const int b = base + threadIdx.x;
        w = b < a.batch ? work_of(seq_of(a, b), a) : 0;
        incl = block_scan(w, sh, sum);
        total += sum;
    }
    Ranges r;
    r.total = total;
    const int64_t want = a.whole_units ? total : (total + kMinTiles - 1) / kMinTiles;
    r.ctas = (int)(want < N * gridDim.x ? want : N * gridDim.x);
    if (c >= r.ctas) return r;
    r.share = quotient(total, r.ctas);
    r.more = (int)(total - r.share * r.ctas);
    auto look = [&](int b) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t target = r.start(c + i);
            if (c + i < r.ctas && target >= incl - w && target < incl) sh_place[i] = Place{b, target - (incl - w)};
        }
    };
    if (a.batch <= kThreads) {
        look(threadIdx.x);
    } else {
        int64_t before = 0;
        for (int base = 0; base < a.batch; base += kThreads) {
            const int b = base + threadIdx.x;
            w = b < a.batch ? work_of(seq_of(a, b), a) : 0;
            incl = block_scan(w, sh, sum) + before;
            look(b);
            before += sum;
        }
    }
    __syncthreads();
    return r;
}

// A block's way through its range, one segment (a unit's tiles t0 .. t1 - 1) after another.
struct Walk {
    Seq s;
    int b, u, t0, t1;
    int64_t pos, end;
    bool whole;
    __device__ __forceinline__ void clip() { t1 = whole ? s.tiles : (int)min((int64_t)s.tiles, t0 + (end - pos)); }
    __device__ __forceinline__ void begin(const KvAttnArgs& a, const Place& p, int64_t first, int64_t last) {
        b = p.b;
        s = seq_of(a, b);
        pos = first;
        end = last;
        whole = a.whole_units;
        u = whole ? (int)p.off : (int)quotient(p.off, s.tiles);
        t0 = whole ? 0 : (int)(p.off - (int64_t)u * s.tiles);
        clip();
    }
    __device__ __forceinline__ bool done() const { return pos >= end; }
    __device__ __forceinline__ void advance(const KvAttnArgs& a) {
        pos += whole ? 1 : t1 - t0;
        if (pos >= end) return;
        if (++u == s.units) {
            u = 0;
            do {
                s = seq_of(a, ++b);
            } while (s.units == 0);
        }
        t0 = 0;
        clip();
    }
};

// ---------------------------------------------------------------- results
// `n` consecutive output values of one row, d .. d + n - 1 (all inside hd): joined with the added pieces, then written.
template <int N>
__device__ __forceinline__ void finish(const KvAttnArgs& a, int64_t row, int head, int d, float m, float l, float (&o)[N]) {
    for (int s = 0; s < a.add.pieces; ++s) {
        const int64_t i = ((int64_t)s * a.M + row) * a.heads + head;
        const float mi = a.add.m[i], li = a.add.l[i], mn = fmaxf(m, mi);
        const float x = m == -INFINITY ? 0.0f : ex2(__fsub_rn(m, mn)), y = mi == -INFINITY ? 0.0f : ex2(__fsub_rn(mi, mn));
        l = __fmaf_rn(l, x, __fmul_rn(li, y));
        const float* p = a.add.o + i * a.c.hd + d;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + j);
            o[j] = __fmaf_rn(o[j], x, __fmul_rn(v.x, y));
            o[j + 1] = __fmaf_rn(o[j + 1], x, __fmul_rn(v.y, y));
            o[j + 2] = __fmaf_rn(o[j + 2], x, __fmul_rn(v.z, y));
            o[j + 3] = __fmaf_rn(o[j + 3], x, __fmul_rn(v.w, y));
        }
        m = mn;
    }
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = l == 0.0f ? 0.0f : __fmul_rn(o[j], inv);
    const int64_t at = row * a.ldo + (int64_t)head * a.c.hd + d;
    if (a.bf16) {
        uint32_t w[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
        __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.o) + at;
        if (N == 8)
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[N / 2 - 2], w[N / 2 - 1]);
        else
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
        float* p = static_cast<float*>(a.o) + at;
#pragma unroll
        for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
    }
}

// ---------------------------------------------------------------- the pass over the keys
// SOLO: a unit's tiles belong to one warp, and nothing is joined.
template <int HD, bool E4M3, bool PREFIX, bool SOLO>
__global__ void __launch_bounds__(kThreads, kPerSm) kv_attention_kernel(const KvAttnArgs a) {
    constexpr int kChunks = HD / 16;          // 16-byte chunks of a code row
    constexpr int kStage = kStageBytes<HD>;
    constexpr int kWords = HD / 16;           // 4-byte words of a thread's share of a key row (MMA k steps of scores)
    constexpr int kVw = HD / 32;              // words of a thread's share of a value row
    constexpr int kNt = HD / 8;               // output n tiles
    constexpr int kOstride = HD / 4 + 4, kOrow = 4 * kOstride;  // padded output rows in shared memory (floats)
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t sh_scan[kWarps];
    constexpr int kTeam = SOLO ? 1 : kWarps, kTeams = kWarps / kTeam;  // warps that share a unit's tiles
    __shared__ Place sh_place[kTeams];
    __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
    __shared__ Walk sh_load[kWarps], sh_walk[kTeams][2];
    __shared__ int sh_free[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    griddep_wait();
    griddep_launch();

    const int team = SOLO ? warp : 0, member = SOLO ? 0 : warp, worker = blockIdx.x * kTeams + team;
    auto sync = [&]() {
        if (SOLO)
            __syncwarp();
        else
            __syncthreads();
    };
    const Ranges rg = find_range(a, blockIdx.x * kTeams, sh_scan, sh_place);
    Border* border = reinterpret_cast<Border*>(a.part + (int64_t)2 * kMaxCtas * kPart<128>) + blockIdx.x;
    if (worker >= rg.ctas) {
        if (!SOLO && threadIdx.x == 0) border->pieces = 0;
        return;
    }
    const int64_t first = rg.start(worker), last = rg.start(worker + 1);
    uint8_t* ring = smem + warp * (kStages * kStage);
    const uint32_t ring_u = smem_u32(ring);

    // The way through the range is kept in shared memory: for each warp's loader, which runs ahead, and (two slots in turn)
    // for the block. Registers hold what a tile needs.
    if (lane == 0) {
        Walk w;
        w.begin(a, sh_place[team], first, last);
        sh_load[warp] = w;
        if (member == 0) sh_walk[team][0] = w;
    }
    sync();

    // ---- loader: the warp's tiles in order, one ahead with the page numbers
    int lt, lt_end, l_len, l_head, l_seq;
    auto take_load = [&]() {
        const Walk& w = sh_load[warp];
        lt = w.t0 + member;
        lt_end = w.t1;
        l_len = w.s.len;
        l_head = w.u / w.s.row_tiles;
        l_seq = w.b;
    };
    take_load();
    int page_a = 0, page_b = 0;
    bool have = true;
    auto fetch = [&]() {  // the next tile of this warp, and the pages of its two halves
        while (lt >= lt_end) {
            __syncwarp();
            if (lane == 0) sh_load[warp].advance(a);
            __syncwarp();
            if (sh_load[warp].done()) {
                have = false;
                return;
            }
            take_load();
        }
        const int k0 = lt * kTile;
        const bool own = !PREFIX || k0 >= a.prefix_pad;
        const int32_t* pg = own ? a.pages + (int64_t)l_seq * a.ld_pages : a.prefix_pages;
        const int k = PREFIX && own ? k0 - a.prefix_pad : k0;
        const int end = !PREFIX ? l_len : own ? l_len - a.prefix_pad : a.prefix_len;
        page_a = k < end ? pg[k >> a.c.page_shift] : 0;
        page_b = k + 16 < end ? pg[(k + 16) >> a.c.page_shift] : 0;
    };
    auto issue = [&](int stage) {
        if (have) {
            const uint32_t st = ring_u + stage * kStage;
            const int at = lt * kTile, k0 = PREFIX && at >= a.prefix_pad ? at - a.prefix_pad : at;  // in the own keys or the prefix
            const int left = (!PREFIX || at >= a.prefix_pad ? l_len : a.prefix_len) - at, mask = (1 << a.c.page_shift) - 1;
            const int h = l_head;
            const bool ok_a = page_a >= 0 && page_a < a.c.n_pages, ok_b = page_b >= 0 && page_b < a.c.n_pages;
            if (!(ok_a && ok_b) && lane == 0) atomicOr(&g_device_error, kErrIndex);
            uint32_t bits = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;  // keys there
            if (!ok_a) bits &= 0xffff0000u;
            if (!ok_b) bits &= 0x0000ffffu;
            // cache rows of keys k0 and (less 16) k0 + 16
            const int64_t ra = (((int64_t)page_a * a.c.kv_heads + h) << a.c.page_shift) + (k0 & mask);
            const int64_t rb = (((int64_t)page_b * a.c.kv_heads + h) << a.c.page_shift) + ((k0 + 16) & mask) - 16;
            constexpr int kRowsAtOnce = 32 / kChunks;
            const int r0 = lane / kChunks, c = lane % kChunks;
            const int64_t offa = (ra + r0) * a.c.hd + c * 16, offb = (rb + r0) * a.c.hd + c * 16;
            const uint32_t mine = c * 16 < a.c.hd ? bits >> r0 : 0u;
            if (bits == 0xffffffffu && a.c.hd == HD) {  // a whole tile: four pointers and constant steps
                const uint8_t *ka = a.c.k + offa, *kb = a.c.k + offb, *va = a.c.v + offa, *vb = a.c.v + offb;
#pragma unroll
                for (int p = 0; p < kTile / kRowsAtOnce; ++p) {
                    const int r = p * kRowsAtOnce + r0, f = HD == 128 ? (r & 7) : ((r >> 1) & 3);
                    const uint32_t dst = st + r * HD + ((c ^ f) << 4);
                    cp_async16(dst, (p * kRowsAtOnce < 16 ? ka : kb) + p * kRowsAtOnce * HD);
                    cp_async16(dst + kTile * HD, (p * kRowsAtOnce < 16 ? va : vb) + p * kRowsAtOnce * HD);
                }
            } else
#pragma unroll
            for (int p = 0; p < kTile / kRowsAtOnce; ++p) {
                const int r = p * kRowsAtOnce + r0;
                const bool on = (mine >> (p * kRowsAtOnce)) & 1;
                const int64_t off = on ? (p * kRowsAtOnce < 16 ? offa : offb) + p * kRowsAtOnce * a.c.hd : 0;
                const int f = HD == 128 ? (r & 7) : ((r >> 1) & 3);
                const uint32_t dst = st + r * HD + ((c ^ f) << 4);
                cp_async16(dst, a.c.k + off, on);
                cp_async16(dst + kTile * HD, a.c.v + off, on);
            }
            const bool on = (bits >> lane) & 1;
            const int64_t row = on ? (lane < 16 ? ra : rb) + lane : 0;
            cp_async4(st + 2 * kTile * HD + lane * 4, a.c.ks + row, on);
            cp_async4(st + 2 * kTile * HD + kTile * 4 + lane * 4, a.c.vs + row, on);
            if (lane == 0) *reinterpret_cast<uint32_t*>(ring + stage * kStage + 2 * kTile * HD + 2 * kTile * 4) = bits;
            lt += kTeam;
            fetch();
        }
        cp_commit();
    };
    if (!SOLO && threadIdx.x == 0) {
        const Walk& cw = sh_walk[0][0];
        Border bd{0, 0, 0, 0, 0, 0};
        if (cw.t0 > 0) {  // this block's start cuts a unit
            const int64_t unit = first - cw.t0, before = rg.start(blockIdx.x - 1);
            if (before <= unit) {  // and no block's before it does
                const int h = cw.u / cw.s.row_tiles;
                bd.pieces = rg.owner(unit + cw.s.tiles - 1) - (int)blockIdx.x + 2;
                bd.slot = before == unit ? 0 : 1;
                bd.lo = cw.s.lo;
                bd.head0 = h * a.group;
                bd.row0 = (cw.u - h * cw.s.row_tiles) * kRows;
                bd.rows = min(kRows, cw.s.n * a.group - bd.row0);
            }
        }
        *border = bd;
    }
    fetch();
    int it = 0;  // tiles this warp has taken

    for (int seg = 0; !sh_walk[team][seg & 1].done(); ++seg) {
        const bool head_seg = seg == 0;
        const Walk& cw = sh_walk[team][seg & 1];
        const int h = cw.u / cw.s.row_tiles, row0 = (cw.u - h * cw.s.row_tiles) * kRows;
        const int rows = min(kRows, cw.s.n * a.group - row0), seg_end = cw.t1;
        // ---- the query row of this thread's group: its share [t * HD / 4, (t + 1) * HD / 4), as fp32 words
        uint4 q[kWords];
        {
            const int r = row0 + min(g, rows - 1), i = a.by_group(r);
            const int64_t at = (cw.s.lo + (int64_t)i) * a.ldq + (int64_t)(h * a.group + (r - i * a.group)) * a.c.hd + t * (HD / 4);
            if (a.bf16) {
#pragma unroll
                for (int j = 0; j < kWords / 2; ++j) {
                    uint4 u = make_uint4(0, 0, 0, 0);
                    if (t * (HD / 4) + 8 * j < a.c.hd) u = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + at)[j];
                    q[2 * j] = make_uint4(u.x << 16, u.x & 0xffff0000u, u.y << 16, u.y & 0xffff0000u);
                    q[2 * j + 1] = make_uint4(u.z << 16, u.z & 0xffff0000u, u.w << 16, u.w & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kWords; ++j) {
                    q[j] = make_uint4(0, 0, 0, 0);
                    if (t * (HD / 4) + 4 * j < a.c.hd) q[j] = reinterpret_cast<const uint4*>(static_cast<const float*>(a.q) + at)[j];
                }
            }
        }
        if (head_seg) {  // the rows are on their way while the pages of the first tiles are waited for
#pragma unroll
            for (int s = 0; s < kStages - 1; ++s) issue(s);
        }
        // ---- as MMA fragments: word w holds hd values 4 w .. 4 w + 3 of the thread's share
        uint32_t qf[kWords][E4M3 ? 4 : 3];  // e4m3: hi, lo of two pairs; int8: three bytes of each value, largest first
        // keys that the row sees: the whole prefix and its own
        const int limit = g >= rows ? 0 : a.causal ? max(PREFIX ? a.prefix_pad : 0, cw.s.len - cw.s.n + a.by_group(row0 + g) + 1) : cw.s.len;
        float rf;  // takes scores back to log2 units
        {
            uint32_t bits = 0;  // of the row's largest |q|
#pragma unroll
            for (int w = 0; w < kWords; ++w)
                bits = max(max(max(bits, q[w].x & 0x7fffffffu), q[w].y & 0x7fffffffu), max(q[w].z & 0x7fffffffu, q[w].w & 0x7fffffffu));
            bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
            bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
            float mul;
            if (E4M3) {  // the row's largest element goes to [2^14, 2^15)
                const int up = min(253, 268 - (int)(bits >> 23));
                mul = pow2_biased(up);
                rf = __fmul_rn(pow2_biased(254 - up), a.scale_log2e);
            } else {  // to 8355000: three signed bytes hold 8355711
                const float big = fmaxf(__uint_as_float(bits), 0x1p-100f);
                mul = __fdiv_rn(8355000.0f, big);
                rf = __fmul_rn(__fdiv_rn(big, 8355000.0f), a.scale_log2e);
            }
            if (bits >= 0x7f800000u) rf = __int_as_float(0x7fc00000);  // an infinity or a NaN makes the row NaN
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                const float y[4] = {__fmul_rn(__uint_as_float(q[w].x), mul), __fmul_rn(__uint_as_float(q[w].y), mul),
                                    __fmul_rn(__uint_as_float(q[w].z), mul), __fmul_rn(__uint_as_float(q[w].w), mul)};
                if constexpr (E4M3) {  // in the order of unpack4's pairs
                    split_h2(y[0], y[1], qf[w][0], qf[w][1]);
                    split_h2(y[2], y[3], qf[w][2], qf[w][3]);
                } else {
                    int v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = __float2int_rn(y[k]);
#pragma unroll
                    for (int part = 2; part >= 0; --part) {
                        const uint32_t ab = __byte_perm(v[0], v[1], 0x0040), cd = __byte_perm(v[2], v[3], 0x0040);
                        qf[w][part] = __byte_perm(ab, cd, 0x5410);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = (v[k] + 128) >> 8;  // what is left above a signed byte
                    }
                }
            }
        }
        float oacc[kNt][4];
#pragma unroll
        for (int n = 0; n < kNt; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) oacc[n][k] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        int vref = 15;  // biased exponent above every value scale so far

        for (int tile = cw.t0 + member; tile < seg_end; tile += kTeam, ++it) {
            cp_wait<kStages - 2>();
            __syncwarp();
            issue((it + kStages - 1) % kStages);
            const uint8_t* st = ring + (it % kStages) * kStage;
            const float* ks = reinterpret_cast<const float*>(st + 2 * kTile * HD);
            const float* vs = ks + kTile;
            const uint32_t there = *reinterpret_cast<const uint32_t*>(vs + kTile);
            // ---- scores of 32 keys: thread (g, t) gets keys 8 n + 2 t, 8 n + 2 t + 1 of row g
            float s[4][2];
            float mx = -INFINITY, vmax = 0.0f;
            float2 vsc[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float s0, s1;  // products of the row with keys 2 t and 2 t + 1
                const int r = n * 8 + g;
                const uint8_t* kr = st + r * HD;
                uint32_t w[kWords];
#pragma unroll
                for (int half = 0; half < kWords / 4; ++half) {
                    const int ch = HD == 128 ? (2 * t + half) ^ (r & 7) : t ^ ((r >> 1) & 3);
                    const uint4 u = *reinterpret_cast<const uint4*>(kr + (ch << 4));
                    w[4 * half] = u.x, w[4 * half + 1] = u.y, w[4 * half + 2] = u.z, w[4 * half + 3] = u.w;
                }
                if constexpr (E4M3) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < kWords; ++k) {
                        uint32_t b0, b1;
                        unpack4<E4M3>(w[k], b0, b1);
                        mma_f16(c, qf[k][0], qf[k][1], qf[k][2], qf[k][3], b0, b1);
                    }
                    s0 = __fadd_rn(c[0], c[2]);
                    s1 = __fadd_rn(c[1], c[3]);
                } else {
                    int c[4] = {0, 0, 0, 0}, d[4] = {0, 0, 0, 0};  // first and second bytes; third bytes
#pragma unroll
                    for (int k = 0; k < kWords; k += 2) {
                        mma_s8(c, qf[k][0], qf[k][1], qf[k + 1][0], qf[k + 1][1], w[k], w[k + 1]);
                        mma_s8(d, qf[k][2], 0u, qf[k + 1][2], 0u, w[k], w[k + 1]);
                    }
                    s0 = __fmaf_rn((float)(c[0] * 256 + c[2]), 256.0f, (float)d[0]);
                    s1 = __fmaf_rn((float)(c[1] * 256 + c[3]), 256.0f, (float)d[1]);
                }
                const float2 f = *reinterpret_cast<const float2*>(ks + n * 8 + 2 * t);
                vsc[n] = *reinterpret_cast<const float2*>(vs + n * 8 + 2 * t);
                const int key = tile * kTile + n * 8 + 2 * t;
                const uint32_t here = there >> (n * 8 + 2 * t);
                const bool see0 = (here & 1) && key < limit, see1 = (here & 2) && key + 1 < limit;
                s[n][0] = see0 ? __fmul_rn(__fmul_rn(s0, f.x), rf) : -INFINITY;
                s[n][1] = see1 ? __fmul_rn(__fmul_rn(s1, f.y), rf) : -INFINITY;
                mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
                // a value scale that a row does not see may be anything
                vsc[n].x = see0 ? vsc[n].x : 0.0f;
                vsc[n].y = see1 ? vsc[n].y : 0.0f;
                vmax = fmaxf(vmax, fmaxf(fabsf(vsc[n].x), fabsf(vsc[n].y)));
            }
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {  // a row's keys are spread over four lanes
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
            }
            // ---- running maximum, and the references that the outputs are kept in
            const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.0f : mn;
            float alpha = m == -INFINITY ? 0.0f : ex2(__fsub_rn(m, mu));
            l = __fmul_rn(l, alpha);
            const int e = __float_as_int(vmax) >> 23;
            bool move = mn != m;
            if (e >= vref) {  // the same in the row's four lanes
                const int nref = min(e + 1, 255);
                alpha = __fmul_rn(alpha, nref - vref > 126 ? 0.0f : pow2_biased(127 - (nref - vref)));
                vref = nref;
                move = true;
            }
            m = mn;
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int n = 0; n < kNt; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) oacc[n][k] = __fmul_rn(oacc[n][k], alpha);
            }
            const float vmul = pow2_biased(268 - vref);
            // ---- probabilities as the A fragments of two 16-key steps
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float p0 = ex2(__fsub_rn(s[n][0], mu)), p1 = ex2(__fsub_rn(s[n][1], mu));
                l = __fadd_rn(l, __fadd_rn(p0, p1));
                split_h2(__fmul_rn(p0, __fmul_rn(vsc[n].x, vmul)), __fmul_rn(p1, __fmul_rn(vsc[n].y, vmul)), ph[n], pl[n]);
            }
            // ---- outputs: n tile j holds hd columns g' * kNt + j
            const uint8_t* vt = st + kTile * HD;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[4][kVw];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = j * 16 + 2 * t + (k & 1) + 8 * (k >> 1);
                    if (HD == 128) {
                        const uint4 u = *reinterpret_cast<const uint4*>(vt + r * HD + ((g ^ (r & 7)) << 4));
                        w[k][0] = u.x, w[k][1] = u.y, w[k][kVw - 2] = u.z, w[k][kVw - 1] = u.w;
                    } else {
                        const uint2 u =
                            *reinterpret_cast<const uint2*>(vt + r * HD + (((g >> 1) ^ ((r >> 1) & 3)) << 4) + (g & 1) * 8);
                        w[k][0] = u.x, w[k][1] = u.y;
                    }
                }
#pragma unroll
                for (int q = 0; q < kVw; ++q) {
                    uint32_t b0[4], b1[4];  // pairs (key 2t, key 2t + 1) and (key 2t + 8, key 2t + 9) of four columns
                    constexpr uint32_t kLo = E4M3 ? 0x5140 : 0x5410, kHi = E4M3 ? 0x7362 : 0x7632;
                    unpack4<E4M3>(__byte_perm(w[0][q], w[1][q], kLo), b0[0], b0[1]);
                    unpack4<E4M3>(__byte_perm(w[0][q], w[1][q], kHi), b0[2], b0[3]);
                    unpack4<E4M3>(__byte_perm(w[2][q], w[3][q], kLo), b1[0], b1[1]);
                    unpack4<E4M3>(__byte_perm(w[2][q], w[3][q], kHi), b1[2], b1[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_f16(oacc[4 * q + k], ph[2 * j], pl[2 * j], ph[2 * j + 1], pl[2 * j + 1], b0[k], b1[k]);
                }
            }
        }

        // ---- join the unit's warps: every warp's free ring stage holds its outputs (the stage that its next copy fills)
        l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 1));
        l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 2));
        if (t == 0) {
            sh_m[warp][g] = m;
            sh_l[warp][g] = l;
        }
        const int free_stage = (it + kStages - 1) % kStages;
        __syncwarp();
        {
            const float back = pow2_biased(vref - 14);
            float* ob = reinterpret_cast<float*>(ring + free_stage * kStage) + g * kOrow + t * kOstride;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int n = 0; n < kNt; n += 4) {
                    float4 x;
                    float* xp = &x.x;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        xp[k] = __fmul_rn(__fadd_rn(oacc[n + k][half], oacc[n + k][2 + half]), back);
                    *reinterpret_cast<float4*>(ob + half * kNt + n) = x;
                }
        }
        if (lane == 0) sh_free[warp] = free_stage;
        if (member == 0 && lane == 0) {  // the next segment; everybody reads it behind the last barrier of this one
            Walk w = cw;
            w.advance(a);
            sh_walk[team][(seg + 1) & 1] = w;
        }
        sync();
#pragma unroll 1
        for (int row = SOLO ? lane / 16 : threadIdx.x / 16; row < kRows; row += 2 * kTeam) {
            constexpr int N = HD / 16;
            const int d = (threadIdx.x % 16) * N;
            float mm = -INFINITY, ll = 0.0f, o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = 0.0f;
#pragma unroll
            for (int w = team; w < team + kTeam; ++w) mm = fmaxf(mm, sh_m[w][row]);
#pragma unroll 1
            for (int w = team; w < team + kTeam; ++w) {
                const float mw = sh_m[w][row], f = mw == -INFINITY ? 0.0f : ex2(__fsub_rn(mw, mm));
                const float* ob = reinterpret_cast<const float*>(smem + (w * kStages + sh_free[w]) * kStage) + row * kOrow +
                                  (d / (HD / 4)) * kOstride + d % (HD / 4);
                ll = __fmaf_rn(sh_l[w][row], f, ll);
#pragma unroll
                for (int j = 0; j < N; ++j) o[j] = __fmaf_rn(ob[j], f, o[j]);
            }
            if (SOLO || (cw.t0 == 0 && cw.t1 == cw.s.tiles)) {
                if (row < rows && d < a.c.hd) {
                    const int r = row0 + row, i = a.by_group(r);
                    finish<N>(a, cw.s.lo + (int64_t)i, h * a.group + (r - i * a.group), d, mm, ll, o);
                }
            } else {  // the first segment goes to slot 0, the last one to slot 1: no other can be cut
                float* p = a.part + ((int64_t)blockIdx.x * 2 + (head_seg ? 0 : 1)) * kPart<HD>;
#pragma unroll
                for (int j = 0; j < N; j += 4)
                    *reinterpret_cast<float4*>(p + row * HD + d + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                if (d == 0) {
                    p[kRows * HD + row] = mm;
                    p[kRows * HD + kRows + row] = ll;
                }
            }
        }
        sync();
    }
    cp_wait<0>();
}

// Joins the partial results of every unit that the borders between blocks cut: block c acts on border c + 1, if it is the
// first one inside its unit. Four groups of threads take every fourth piece, eight in flight; a long unit may have hundreds.
constexpr int kJoinGroups = 4, kJoinThreads = kThreads * kJoinGroups;
template <int HD>
__global__ void __launch_bounds__(kJoinThreads) kv_attention_join_kernel(const KvAttnArgs a) {
    constexpr int N = HD / 16;
    __shared__ float sh_m[kJoinGroups][kRows], sh_l[kJoinGroups][kRows];
    __shared__ __align__(16) float sh_o[kJoinGroups][kRows][HD];
    griddep_wait();
    griddep_launch();
    const int c = blockIdx.x;
    const Border bd = reinterpret_cast<const Border*>(a.part + (int64_t)2 * kMaxCtas * kPart<128>)[c + 1];
    if (bd.pieces == 0) return;
    const int group = threadIdx.x / kThreads, row = threadIdx.x % kThreads / 16, d = (threadIdx.x % 16) * N;
    auto piece = [&](int k) { return a.part + ((int64_t)(c + k) * 2 + (k == 0 ? bd.slot : 0)) * kPart<HD>; };
    float m = -INFINITY, l = 0.0f, o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = 0.0f;
#pragma unroll 8
    for (int k = group; k < bd.pieces; k += kJoinGroups) m = fmaxf(m, piece(k)[kRows * HD + row]);
#pragma unroll 8
    for (int k = group; k < bd.pieces; k += kJoinGroups) {
        const float* p = piece(k);
        const float mk = p[kRows * HD + row], f = mk == -INFINITY ? 0.0f : ex2(__fsub_rn(mk, m));
        l = __fmaf_rn(p[kRows * HD + kRows + row], f, l);
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + row * HD + d + j);
            o[j] = __fmaf_rn(v.x, f, o[j]);
            o[j + 1] = __fmaf_rn(v.y, f, o[j + 1]);
            o[j + 2] = __fmaf_rn(v.z, f, o[j + 2]);
            o[j + 3] = __fmaf_rn(v.w, f, o[j + 3]);
        }
    }
    if (d == 0) {
        sh_m[group][row] = m;
        sh_l[group][row] = l;
    }
#pragma unroll
    for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(&sh_o[group][row][d + j]) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
    __syncthreads();
    if (group != 0 || row >= bd.rows || d >= a.c.hd) return;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoinGroups; ++k) m = fmaxf(m, sh_m[k][row]);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoinGroups; ++k) {
        const float f = sh_m[k][row] == -INFINITY ? 0.0f : ex2(__fsub_rn(sh_m[k][row], m));
        l = __fmaf_rn(sh_l[k][row], f, l);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = __fmaf_rn(sh_o[k][row][d + j], f, o[j]);
    }
    const int r = bd.row0 + row, i = a.by_group(r);
    finish<N>(a, bd.lo + (int64_t)i, bd.head0 + (r - i * a.group), d, m, l, o);
}

int resident_blocks() {
    static std::atomic<int> cache[128];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return kPerSm * 148;
    if (!cache[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cache[dev] = kPerSm * n < kMaxCtas ? kPerSm * n : kMaxCtas;
    }
    return cache[dev];
}

template <typename K>
cudaError_t launch_args(K kernel, int grid, int block, size_t smem, const KvAttnArgs& a, cudaStream_t st) {
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
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int HD, bool E4M3, bool PREFIX>
cudaError_t launch_typed(const KvAttnArgs& a, cudaStream_t st) {
    const size_t smem = (size_t)kWarps * kStages * kStageBytes<HD>;
    const int grid = resident_blocks();
    KvAttnArgs b = a;
    b.prefix_pad = (int)round_up(a.prefix_len, kTile);
    b.whole_units = b.prefix_pad + (a.max_pages << a.c.page_shift) <= kWholeTiles * kTile;
    // units, as far as the host knows: the longer sequences of a mixed batch are not among them
    const int64_t mean = ceil_div(a.M * a.group, a.batch), each = mean > a.max_rows ? 1 : ceil_div(mean, kRows);
    const int64_t tiles = (b.prefix_pad + (a.max_pages << a.c.page_shift)) / kTile;
    const bool solo = b.whole_units && tiles <= kSoloTiles && 8 * each * a.batch * a.c.kv_heads > (8 + tiles) * grid;
    const auto kernel = solo ? kv_attention_kernel<HD, E4M3, PREFIX, true> : kv_attention_kernel<HD, E4M3, PREFIX, false>;
    cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    if ((e = launch_args(kernel, grid, kThreads, smem, b, st)) != cudaSuccess || b.whole_units) return e;
    return launch_args(kv_attention_join_kernel<HD>, grid - 1, kJoinThreads, 0, b, st);
}
template <int HD, bool E4M3>
cudaError_t launch_prefix(const KvAttnArgs& a, cudaStream_t st) {
    return a.prefix_len > 0 ? launch_typed<HD, E4M3, true>(a, st) : launch_typed<HD, E4M3, false>(a, st);
}

}  // namespace

size_t kv_attn_part_bytes() { return sizeof(float) * 2 * kMaxCtas * kPart<128> + sizeof(Border) * (kMaxCtas + 1); }

cudaError_t launch_kv_attention(const KvAttnArgs& a, cudaStream_t st) {
    if (a.batch <= 0 || a.M <= 0) return cudaSuccess;
    if (a.c.hd > 64) return a.c.e4m3 ? launch_prefix<128, true>(a, st) : launch_prefix<128, false>(a, st);
    return a.c.e4m3 ? launch_prefix<64, true>(a, st) : launch_prefix<64, false>(a, st);
}

}  // namespace b2s
