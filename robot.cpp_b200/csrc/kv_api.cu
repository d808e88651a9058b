// kv_api.cu -- the extern "C" boundary of include/b2s_kv.h: argument checks, workspace layout, dispatch.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "b2s_internal.h"
#include "b2s_kv.h"
#include "kv_internal.h"

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return b2s::set_last_error(code, buf);
}

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return B2S_OK;
    (void)cudaGetLastError();  // a failed launch must not leak into the next call's error check
    return fail(B2S_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t a256(size_t v) { return (v + 255) & ~size_t(255); }
constexpr int64_t kMaxInt = 0x7fffffff;
constexpr int kMaxBatch = 16384;

int check_type(int32_t type, const char* op) {
    if (type != B2S_TYPE_F32 && type != B2S_TYPE_BF16)
        return fail(B2S_ERR_UNSUPPORTED, "%s: type %d is not f32 or bf16", op, (int)type);
    return B2S_OK;
}
size_t size_of(int32_t type) { return type == B2S_TYPE_BF16 ? 2 : 4; }

// M rows of `width` values of `type`, 16-byte aligned.
int check_rows(const void* p, int64_t M, int64_t ld, int64_t width, int32_t type, const char* op, const char* name) {
    if (M == 0) return B2S_OK;
    if (!p) return fail(B2S_ERR_INVALID_ARG, "%s: %s is NULL", op, name);
    if (ld < width) return fail(B2S_ERR_INVALID_ARG, "%s: %s rows of %lld values have stride %lld", op, name, (long long)width, (long long)ld);
    if (!aligned(p, 16) || ld * (int64_t)size_of(type) % 16 != 0)
        return fail(B2S_ERR_UNSUPPORTED, "%s: %s needs a 16-byte aligned base and a row stride that is a multiple of 16 bytes", op, name);
    return B2S_OK;
}

int cache_view(const b2s_kv_cache* c, b2s::KvView* v, const char* op) {
    if (!c) return fail(B2S_ERR_INVALID_ARG, "%s: cache is NULL", op);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(B2S_ERR_INVALID_ARG, "%s: a cache buffer is NULL", op);
    if (c->type != B2S_TYPE_I8 && c->type != B2S_TYPE_F8_E4M3)
        return fail(B2S_ERR_UNSUPPORTED, "%s: cache type %d is not i8 or f8_e4m3", op, (int)c->type);
    if (c->n_kv_heads <= 0 || c->head_dim <= 0 || c->n_pages <= 0 || c->page_size <= 0)
        return fail(B2S_ERR_INVALID_ARG, "%s: cache has a non-positive dimension", op);
    if (c->head_dim % 16 != 0 || c->head_dim > 128)
        return fail(B2S_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 16 up to 128", op, c->head_dim);
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return fail(B2S_ERR_UNSUPPORTED, "%s: page_size %d is not a power of two from 16 to 1024", op, c->page_size);
    if (c->n_kv_heads > 4096 || c->n_pages > kMaxInt)
        return fail(B2S_ERR_UNSUPPORTED, "%s: cache of %d heads and %lld pages is too large", op, c->n_kv_heads, (long long)c->n_pages);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(B2S_ERR_UNSUPPORTED, "%s: cache codes need 16-byte alignment, scales 4-byte", op);
    v->k = static_cast<uint8_t*>(c->k);
    v->v = static_cast<uint8_t*>(c->v);
    v->ks = c->k_scale;
    v->vs = c->v_scale;
    v->n_pages = c->n_pages;
    v->kv_heads = c->n_kv_heads;
    v->hd = c->head_dim;
    v->page_shift = __builtin_ctz((unsigned)c->page_size);
    v->e4m3 = c->type == B2S_TYPE_F8_E4M3;
    return B2S_OK;
}

// Which kernels take the rows of a call, decided from sizes that the host has. Sequences with at most kFewRows rows a
// key/value head go to the warp-level kernel, which reads their keys once per eight rows; the others to the tensor-core
// kernel, which reads them once per 128. Five heads of 128, int8, us with the first and with the second kernel: 16 sequences
// of 2000 keys, 20 rows 40 and 60 (bf16 39 and 56), 32 rows 48 and 62 (46 and 56), 48 rows 64 and 62 (63 and 58), 64 rows 81 and
// 65 (79 and 59); one sequence, 32 rows 18.5 and 20.0 (17.0 and 18.1), 64 rows 21.6 and 20.8 (20.2 and 18.9).
constexpr int kFewRows = 32;
struct Plan {
    bool few, many, pair;  // pair: blocks of 256 rows
    int min_rows, splits;
};
// The tensor-core kernel's part of a plan for M tokens of up to max_q a sequence over `keys` keys: blocks of 128 or (bf16) 256
// rows, and into how many shares the keys are cut where that gives less than a wave of blocks. The least estimate is taken, in
// half tiles' time: waves x (a block's tiles of 128 keys, 2 each or 3 for 256 rows, + 8 or 12 to start and end it), + 6 for the
// join. bf16, five heads, us with blocks of 128 and of 256 rows: one sequence of 256 rows on 2000 keys 22 and 28, 8 of 260 on
// 2000 keys 58 and 83, 2 of 2048 on 4096 keys 173 and 141, 8 of 512 on 128 keys 26 and 19. fp32, whole keys and cut ones: 260
// rows on 8192 keys 183 and 44, 512 on 2000 keys 59 and 29, 4096 rows of one head on 4096 keys 100 and 45. The host knows the
// table's width, not the lengths in it: 4 sequences of 100 fp32 tokens take 17 us behind a table of 2 pages of 64 and 45 behind
// one of 128, whose keys are cut for nothing.
constexpr int kMaxSplits = 16, kWave = 148;
int64_t waves(int64_t units, int s) { return (units * s + kWave - 1) / kWave; }
constexpr int tile_cost(int pair) { return 2 + pair; }
constexpr int block_cost(int pair) { return 8 + 4 * pair; }
constexpr int kJoinCost = 6;
void plan_blocks(Plan* p, int64_t M, int64_t max_q, int group, int kv_heads, int64_t keys, bool bf16) {
    p->many = true;
    const int64_t seqs = (M + max_q - 1) / max_q, tiles = std::max<int64_t>(1, (keys + 127) / 128);
    int64_t best = -1;
    for (int pair = 0; pair <= (bf16 ? 1 : 0); ++pair) {
        const int64_t units = std::max<int64_t>(1, seqs) * ((max_q * group + 128 * (1 + pair) - 1) / (128 * (1 + pair))) * kv_heads;
        for (int s = 1; s <= kMaxSplits && s <= tiles && (s == 1 || units < kWave); ++s) {
            const int64_t cost = waves(units, s) * ((tiles + s - 1) / s * tile_cost(pair) + block_cost(pair)) + (s > 1 ? kJoinCost : 0);
            if (best < 0 || cost < best) {
                best = cost;
                p->pair = pair != 0;
                p->splits = s;
            }
        }
    }
}
// Whether a call of `units` blocks over some number of tiles up to `most` may be cut into s shares: that has to cost less than
// every smaller number, s1, of them, tiles / s tiles a share and without rounding up against (tiles + s1 - 1) / s1. Both sides are
// linear in the tiles, so where it is false for the fewest and for the most tiles it is false between them.
bool may_be_cut(int64_t units, int s, int64_t most, int pair) {
    const int64_t w = waves(units, s), tile = tile_cost(pair), block = block_cost(pair);
    for (int s1 = 1; s1 < s; ++s1) {
        const int64_t w1 = waves(units, s1);
        auto less = [&](int64_t tiles) {  // times s s1
            return s1 * (w * (tile * tiles + block * s) + kJoinCost * s) <
                   s * (w1 * (tile * (tiles + s1 - 1) + block * s1) + (s1 > 1 ? kJoinCost * s1 : 0));
        };
        if (!less(s) && !less(most)) return false;
    }
    return true;
}
// A bound of the pieces (of a row and head) that cut keys leave in any call of up to `rows` rows x heads over up to `keys` keys:
// calls of fewer rows or keys may be cut where the largest is not. A call of `units` < kWave blocks has at most that many times 128
// or 256 rows x heads.
int64_t most_pieces(int64_t rows, int kv_heads, int64_t keys) {
    int64_t most = 0;
    const int64_t tiles = (keys + 127) / 128;
    for (int64_t units = kv_heads; units < kWave; units += kv_heads)
        for (int pair = 0; pair < 2; ++pair) {
            const int64_t held = std::min(rows, units * 128 * (1 + pair));
            for (int s = (int)std::min<int64_t>(kMaxSplits, tiles); s > 1 && held * s > most; --s)
                if (may_be_cut(units, s, tiles, pair)) most = held * s;
        }
    return most;
}
Plan plan_rows(int64_t M, int64_t batch, int64_t max_q, int group, int kv_heads, int64_t keys, bool bf16) {
    Plan p{true, false, false, 0, 1};
    max_q = std::min(max_q, M);  // it may be any bound
    if (max_q * group <= kFewRows) return p;
    plan_blocks(&p, M, max_q, group, kv_heads, keys, bf16);
    p.few = M != batch * max_q;  // equal: every sequence has max_q rows
    p.min_rows = p.few ? kFewRows : 0;
    return p;
}

// A shared prefix goes through the tensor-core kernel, once for all rows, unless few rows make it cheaper to let every
// sequence read it with its own tokens (from L2): up to kPrefixSteps steps of 32 keys and eight rows. One pass then takes the
// place of three. 20 heads on 5, int8, us with one pass and with three: 16 rows on 545 shared tokens (1440 steps) 21.3 and 25.3,
// 32 on 1600 (8000) 29.6 and 30.7, 64 on 800 (8000) 31.8 and 30.4, 64 on 1600 (16000) 43.1 and 32.5.
constexpr int64_t kPrefixSteps = 8192;
bool prefix_inline(bool own_many, int64_t M, int64_t batch, int64_t max_q, int group, int kv_heads, int64_t prefix_len) {
    return M == 0 || (!own_many && batch * kv_heads * ((std::min(max_q, M) * group + 7) / 8) * ((prefix_len + 31) / 32) <= kPrefixSteps);
}
Plan plan_prefix(const Plan& own, int64_t M, int64_t batch, int64_t max_q, int group, int kv_heads, int64_t prefix_len, bool bf16) {
    Plan p{false, false, false, 0, 1};
    if (prefix_len == 0) return p;
    if (prefix_inline(own.many, M, batch, max_q, group, kv_heads, prefix_len))
        p.few = true;
    else
        plan_blocks(&p, M, M, group, kv_heads, prefix_len, bf16);
    return p;
}

// Workspace of an attention call: partial results, then the softmax states of the own tokens' and the prefix's pieces.
struct StateWs {
    size_t m, l, o;
    int pieces;
};
size_t state_bytes(size_t records, int hd) { return 2 * a256(records * sizeof(float)) + a256(records * hd * sizeof(float)); }
struct AttnWs {
    size_t part, total;
    StateWs own, prefix;
};
AttnWs attn_ws(const Plan& own, const Plan& pre, int64_t M, int heads, int hd) {
    AttnWs w;
    w.part = 0;
    w.total = a256(b2s::kv_attn_part_bytes());
    auto take = [&](int pieces) {
        const size_t rows = (size_t)M * heads * pieces;
        StateWs s;
        s.pieces = pieces;
        s.m = w.total;
        s.l = s.m + a256(rows * sizeof(float));
        s.o = s.l + a256(rows * sizeof(float));
        w.total = s.m + state_bytes(rows, hd);
        return s;
    };
    w.own = take(own.many && (own.splits > 1 || pre.many) ? own.splits : 0);
    w.prefix = take(pre.many ? pre.splits : 0);
    return w;
}

int check_shapes(const b2s::KvView& v, const b2s_kv_batch* b, int64_t M, int n_heads, int64_t prefix_len, const char* op) {
    if (!b) return fail(B2S_ERR_INVALID_ARG, "%s: batch is NULL", op);
    if (b->batch < 0 || M < 0 || b->max_q < 0 || b->max_pages < 0 || prefix_len < 0)
        return fail(B2S_ERR_INVALID_ARG, "%s: a size is negative", op);
    if (n_heads <= 0 || n_heads % v.kv_heads != 0)
        return fail(B2S_ERR_INVALID_ARG, "%s: %d query heads on %d key/value heads", op, n_heads, v.kv_heads);
    if (b->batch > kMaxBatch) return fail(B2S_ERR_UNSUPPORTED, "%s: %d sequences, at most %d", op, b->batch, kMaxBatch);
    const int64_t most = kMaxInt - 1024;
    if (M > most / n_heads || prefix_len > most || b->max_pages > ((most - prefix_len) >> v.page_shift))
        return fail(B2S_ERR_UNSUPPORTED, "%s: rows x heads and prefix_len + tokens of a sequence have to be below 2^31", op);
    return B2S_OK;
}

int attention(const char* op, const b2s_kv_cache* cache, const b2s_kv_batch* batch, const int32_t* prefix_pages,
              int64_t prefix_len, int32_t type, const void* q, int64_t ldq, int64_t M, int n_heads, float scale, int causal,
              void* o, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    b2s::KvView v{};
    int rc;
    if ((rc = cache_view(cache, &v, op))) return rc;
    if ((rc = check_type(type, op))) return rc;
    if ((rc = check_shapes(v, batch, M, n_heads, prefix_len, op))) return rc;
    const int64_t width = (int64_t)n_heads * v.hd;
    if ((rc = check_rows(q, M, ldq, width, type, op, "q"))) return rc;
    if ((rc = check_rows(o, M, ldo, width, type, op, "o"))) return rc;
    if (M > 1 && q == o && ldq != ldo) return fail(B2S_ERR_INVALID_ARG, "%s: in place needs ldq == ldo", op);
    if (!std::isfinite(scale * 2.0f)) return fail(B2S_ERR_INVALID_ARG, "%s: scale is not finite or too large", op);
    if (batch->batch > 0) {
        if (!batch->q_start || !batch->kv_len) return fail(B2S_ERR_INVALID_ARG, "%s: q_start or kv_len is NULL", op);
        if (batch->max_pages > 0 && !batch->pages) return fail(B2S_ERR_INVALID_ARG, "%s: pages is NULL", op);
        if (batch->ld_pages < batch->max_pages) return fail(B2S_ERR_INVALID_ARG, "%s: ld_pages < max_pages", op);
    }
    if (prefix_len > 0 && !prefix_pages) return fail(B2S_ERR_INVALID_ARG, "%s: prefix_pages is NULL", op);
    const int group = n_heads / v.kv_heads;
    const bool bf16 = type == B2S_TYPE_BF16;
    const Plan own = plan_rows(M, batch->batch, batch->max_q, group, v.kv_heads, batch->max_pages << v.page_shift, bf16);
    const Plan pre = plan_prefix(own, M, batch->batch, batch->max_q, group, v.kv_heads, prefix_len, bf16);
    const AttnWs w = attn_ws(own, pre, M, n_heads, v.hd);
    if (!workspace || workspace_bytes < w.total)
        return fail(B2S_ERR_WORKSPACE, "%s needs %zu workspace bytes, got %zu", op, w.total, workspace ? workspace_bytes : 0);
    if (!aligned(workspace, 256)) return fail(B2S_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", op);
    if ((rc = b2s_device_check())) return rc;
    if (M == 0 || batch->batch == 0) return B2S_OK;

    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    b2s::KvAttnArgs a{};
    a.c = v;
    a.q = q;
    a.o = o;
    a.ldq = ldq;
    a.ldo = ldo;
    a.M = M;
    a.heads = n_heads;
    a.group = group;
    while ((1u << a.group_shift) < (uint32_t)group) ++a.group_shift;  // n / group as a multiplication, for n < 2^31
    a.group_mul = (uint32_t)((((uint64_t)1 << 32) * ((1u << a.group_shift) - (uint32_t)group)) / (uint32_t)group + 1);
    a.scale_log2e = scale * 1.4426950408889634f;
    a.bf16 = bf16;
    a.part = reinterpret_cast<float*>(ws + w.part);
    a.q_start = batch->q_start;
    auto state = [&](const StateWs& s) {
        return b2s::AttnState{reinterpret_cast<float*>(ws + s.m), reinterpret_cast<float*>(ws + s.l),
                              reinterpret_cast<float*>(ws + s.o), s.pieces};
    };
    if (pre.many) {  // the batch's rows as one sequence over the prefix
        b2s::KvAttnArgs p = a;
        p.batch = 1;
        p.q_stride = batch->batch;
        p.kv_const = prefix_len;
        p.pages = prefix_pages;
        p.max_pages = (prefix_len + cache->page_size - 1) / cache->page_size;
        p.to_state = true;
        p.out = state(w.prefix);
        if ((rc = launched(b2s::launch_kv_attention_tc(p, pre.pair, pre.splits, st), op))) return rc;
        a.add = p.out;
    }
    a.batch = batch->batch;
    a.q_stride = 1;
    a.kv_len = batch->kv_len;
    a.pages = batch->pages;
    a.ld_pages = batch->ld_pages;
    a.max_pages = batch->max_pages;
    a.causal = causal != 0;
    if (own.many) {
        b2s::KvAttnArgs t = a;
        t.min_rows = own.min_rows;
        t.out = state(w.own);
        t.to_state = w.own.pieces > 0;
        if ((rc = launched(b2s::launch_kv_attention_tc(t, own.pair, own.splits, st), op))) return rc;
        if (t.to_state && (rc = launched(b2s::launch_kv_state_join(t, st), op))) return rc;
    }
    if (!own.few) return B2S_OK;
    a.max_rows = own.many ? kFewRows : (int)kMaxInt;
    if (pre.few) {
        a.prefix_pages = prefix_pages;
        a.prefix_len = (int)prefix_len;
    }
    return launched(b2s::launch_kv_attention(a, st), op);
}

}  // namespace

extern "C" {

int b2s_rope_axes(int32_t type, const void* x, int64_t ldx, int64_t M, int n_heads, int head_dim, const int32_t* pos,
                  int64_t ldpos, int n_axes, const int32_t* sections, int interleaved, float theta_base, void* y,
                  int64_t ldy, void* stream) {
    int rc;
    if ((rc = check_type(type, "rope_axes"))) return rc;
    if (!sections || (M > 0 && (!x || !y || !pos)))
        return fail(B2S_ERR_INVALID_ARG, "rope_axes: x, y, pos and sections must be non-NULL");
    if (M < 0 || n_heads <= 0 || head_dim <= 0 || head_dim % 2) return fail(B2S_ERR_INVALID_ARG, "rope_axes: bad shape");
    const int64_t width = (int64_t)n_heads * head_dim;
    if (head_dim > 256 || M > kMaxInt / n_heads || width / 2 > kMaxInt - 256)  // a row's pairs are counted in 32 bits, 256 a step
        return fail(B2S_ERR_UNSUPPORTED, "rope_axes: head_dim up to 256, M x n_heads and a row's pairs below 2^31");
    if (ldx < width || ldy < width) return fail(B2S_ERR_INVALID_ARG, "rope_axes: row stride below n_heads * head_dim");
    if (!aligned(x, size_of(type)) || !aligned(y, size_of(type)))
        return fail(B2S_ERR_UNSUPPORTED, "rope_axes: x or y is not aligned to its type");
    if (M > 1 && x == y && ldx != ldy) return fail(B2S_ERR_INVALID_ARG, "rope_axes: in place needs ldx == ldy");
    if (n_axes < 1 || n_axes > 4 || ldpos < n_axes) return fail(B2S_ERR_INVALID_ARG, "rope_axes: n_axes must be 1..4 and ldpos >= n_axes");
    if (!(theta_base > 0.0f) || !std::isfinite(theta_base)) return fail(B2S_ERR_INVALID_ARG, "rope_axes: theta_base must be positive");
    int64_t sum = 0;
    for (int i = 0; i < n_axes; ++i) {
        if (sections[i] < 0) return fail(B2S_ERR_INVALID_ARG, "rope_axes: a section is negative");
        sum += sections[i];
    }
    if (sum != head_dim / 2)
        return fail(B2S_ERR_INVALID_ARG, "rope_axes: sections add up to %lld, not to head_dim / 2 = %d", (long long)sum, head_dim / 2);
    b2s::RopePairs p{};
    const int half = head_dim / 2;
    int left[4] = {0, 0, 0, 0};
    for (int i = 0; i < n_axes; ++i) left[i] = sections[i];
    // theta_base^(-2 i / hd) / pi by repeated products in extended precision (their errors stay far below a double's step)
    const long double ratio = std::pow((long double)theta_base, -2.0L / head_dim);
    long double turn = 1.0L / 3.14159265358979323846264338L;
    for (int i = 0, ax = 0; i < half; ++i) {
        while (left[ax] == 0) ax = (ax + 1) % n_axes;
        p.axis[i] = (uint8_t)ax;
        --left[ax];
        if (interleaved) ax = (ax + 1) % n_axes;
        p.turn[i] = (double)turn;
        turn *= ratio;
    }
    if ((rc = b2s_device_check())) return rc;
    return launched(b2s::launch_rope_axes(type == B2S_TYPE_BF16, x, ldx, M, n_heads, head_dim, pos, ldpos, p, y, ldy,
                                          static_cast<cudaStream_t>(stream)),
                    "rope_axes");
}

int b2s_kv_write(const b2s_kv_cache* cache, int32_t type, const void* k, int64_t ldk, const void* v, int64_t ldv,
                 int64_t M, const int64_t* slots, void* stream) {
    b2s::KvView c{};
    int rc;
    if ((rc = cache_view(cache, &c, "kv_write"))) return rc;
    if ((rc = check_type(type, "kv_write"))) return rc;
    if (M < 0) return fail(B2S_ERR_INVALID_ARG, "kv_write: M is negative");
    if (M > kMaxInt / c.kv_heads) return fail(B2S_ERR_UNSUPPORTED, "kv_write: M x n_kv_heads has to be below 2^31");
    if (M > 0 && !slots) return fail(B2S_ERR_INVALID_ARG, "kv_write: slots is NULL");
    const int64_t width = (int64_t)c.kv_heads * c.hd;
    if ((rc = check_rows(k, M, ldk, width, type, "kv_write", "k"))) return rc;
    if ((rc = check_rows(v, M, ldv, width, type, "kv_write", "v"))) return rc;
    if ((rc = b2s_device_check())) return rc;
    return launched(b2s::launch_kv_write(c, type == B2S_TYPE_BF16, k, ldk, v, ldv, M, slots, static_cast<cudaStream_t>(stream)),
                    "kv_write");
}

int b2s_kv_read(const b2s_kv_cache* cache, const int64_t* slots, int64_t M, int32_t type, void* k, int64_t ldk, void* v,
                int64_t ldv, void* stream) {
    b2s::KvView c{};
    int rc;
    if ((rc = cache_view(cache, &c, "kv_read"))) return rc;
    if ((rc = check_type(type, "kv_read"))) return rc;
    if (M < 0) return fail(B2S_ERR_INVALID_ARG, "kv_read: M is negative");
    if (M > kMaxInt / c.kv_heads) return fail(B2S_ERR_UNSUPPORTED, "kv_read: M x n_kv_heads has to be below 2^31");
    if (M > 0 && !slots) return fail(B2S_ERR_INVALID_ARG, "kv_read: slots is NULL");
    if (M > 0 && !k && !v) return fail(B2S_ERR_INVALID_ARG, "kv_read: k and v are both NULL");
    const int64_t width = (int64_t)c.kv_heads * c.hd;
    if (k && (rc = check_rows(k, M, ldk, width, type, "kv_read", "k"))) return rc;
    if (v && (rc = check_rows(v, M, ldv, width, type, "kv_read", "v"))) return rc;
    if ((rc = b2s_device_check())) return rc;
    return launched(b2s::launch_kv_read(c, slots, M, type == B2S_TYPE_BF16, k, ldk, v, ldv, static_cast<cudaStream_t>(stream)),
                    "kv_read");
}

size_t b2s_attention_kv_workspace_size(const b2s_kv_cache* cache, const b2s_kv_batch* batch, int64_t M, int n_heads,
                                       int64_t prefix_len) {
    b2s::KvView v{};
    if (cache_view(cache, &v, "attention_kv_workspace_size")) return 0;
    if (check_shapes(v, batch, M, n_heads, prefix_len, "attention_kv_workspace_size")) return 0;
    // Enough for either type and for every call of no larger sizes: both rules that lead to states hold for the given sizes if they
    // hold for any smaller ones, but how many pieces there are does not grow with the sizes.
    const int group = n_heads / v.kv_heads;
    const int64_t rows = M * n_heads;
    const bool many = std::min<int64_t>(batch->max_q, M) * group > kFewRows;
    const bool shared = prefix_len > 0 && !prefix_inline(many, M, batch->batch, batch->max_q, group, v.kv_heads, prefix_len);
    int64_t own = 0, pre = 0;
    if (many) own = std::max(most_pieces(rows, v.kv_heads, batch->max_pages << v.page_shift), shared ? rows : 0);
    if (shared) pre = std::max(most_pieces(rows, v.kv_heads, prefix_len), rows);
    return a256(b2s::kv_attn_part_bytes()) + state_bytes((size_t)own, v.hd) + state_bytes((size_t)pre, v.hd);
}

int b2s_attention_kv(const b2s_kv_cache* cache, const b2s_kv_batch* batch, int32_t type, const void* q, int64_t ldq,
                     int64_t M, int n_heads, float scale, int causal, void* o, int64_t ldo, void* workspace,
                     size_t workspace_bytes, void* stream) {
    return attention("attention_kv", cache, batch, nullptr, 0, type, q, ldq, M, n_heads, scale, causal, o, ldo, workspace,
                     workspace_bytes, stream);
}

int b2s_attention_kv_prefix(const b2s_kv_cache* cache, const b2s_kv_batch* batch, const int32_t* prefix_pages,
                            int64_t prefix_len, int32_t type, const void* q, int64_t ldq, int64_t M, int n_heads,
                            float scale, int causal, void* o, int64_t ldo, void* workspace, size_t workspace_bytes,
                            void* stream) {
    return attention("attention_kv_prefix", cache, batch, prefix_pages, prefix_len, type, q, ldq, M, n_heads, scale, causal,
                     o, ldo, workspace, workspace_bytes, stream);
}

}  // extern "C"
