// Host side of the paged cache: the handle, its checks, the batch's way to the device, and which kernels a call launches.
// Everything is checked before anything is enqueued.
#include "paged_handle.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <new>

using namespace itak;

namespace {

// Words of a batch on their way to the device travel as the arguments of launches that store them: in the stream's order, with
// no host memory that has to outlive the call.
template <uint32_t N>
struct Words {
    uint32_t *dst;
    uint32_t at0, n0;  // w[0 .. n0) to dst + at0
    uint32_t at1, n1;  // and the n1 behind them to dst + at1
    uint32_t w[N];
};
template <uint32_t N>
__global__ __launch_bounds__(256) void paged_words_kernel(Words<N> a) {
    for (uint32_t i = threadIdx.x; i < a.n0 + a.n1; i += 256) {
        const uint32_t at = i < a.n0 ? a.at0 + i : a.at1 + (i - a.n0);
        a.dst[at] = a.w[i];
    }
}
template <uint32_t N>
void send(uint32_t *dst, uint32_t at0, const uint32_t *w0, uint32_t n0, uint32_t at1, const uint32_t *w1, uint32_t n1,
          hipStream_t stream) {
    Words<N> a;
    a.dst = dst, a.at0 = at0, a.n0 = n0, a.at1 = at1, a.n1 = n1;
    std::copy(w0, w0 + n0, a.w);
    std::copy(w1, w1 + n1, a.w + n0);
    launch_kernel(paged_words_kernel<N>, 1, 256, 0, stream, a);
}
}  // namespace

void itak::send_words(uint32_t *dst, uint32_t at0, const uint32_t *w0, uint32_t n0, uint32_t at1, const uint32_t *w1, uint32_t n1,
                hipStream_t stream) {
    if (n0 + n1 <= kFewWords)
        send<kFewWords>(dst, at0, w0, n0, at1, w1, n1, stream);
    else
        send<kManyWords>(dst, at0, w0, n0, at1, w1, n1, stream);
}

namespace {

itak_status grow(itak_paged *p, void **buffer, uint64_t *have, uint64_t need, const char *what, bool exactly = false) {
    if (need <= *have) return ITAK_OK;
    if (capturing(p->stream))
        return set_error(p->err, ITAK_CAPACITY_EXCEEDED, what, need, *have, 0, 0,
                         "%s: the call needs %llu bytes and the stream is being captured; make the call once uncaptured first", what,
                         ULL(need));
    const uint64_t want = exactly ? need : std::max<uint64_t>(need + need / 2, 1u << 20);
    p->buffers.reserve(p->buffers.size() + 1);
    void *at = nullptr;
    HIP_TRY(p, hipMalloc(&at, want), what);
    p->buffers.push_back(at);
    *buffer = at;
    *have = want;
    return ITAK_OK;
}

uint64_t elem_size(uint32_t elem) { return elem == ITAK_ELEM_F32 ? 4 : 2; }

// The refusals of a configuration; fills geometry and size.
itak_status check_config(ErrorState &e, const itak_paged_config *c, PagedGeom &g, uint64_t &layer_stride, uint64_t &bytes) {
    if (!c) return invalid_argument(e, "config is null");
    if (c->layer_count == 0) return zero_dimension(e, "layer_count");
    if (c->num_kv_heads == 0) return zero_dimension(e, "num_kv_heads");
    if (c->head_dim == 0) return zero_dimension(e, "head_dim");
    if (c->page_count == 0) return zero_dimension(e, "page_count");
    if (c->max_sequences == 0) return zero_dimension(e, "max_sequences");
    if (c->elem != ITAK_ELEM_F16 && c->elem != ITAK_ELEM_BF16)
        return invalid_argument(e, "elem is neither ITAK_ELEM_F16 nor ITAK_ELEM_BF16");
    if (c->head_dim % 8 || c->head_dim > 256) return unsupported(e, "head_dim is no multiple of 8 up to 256");
    if (c->page_rows < 16 || c->page_rows > 1024 || (c->page_rows & (c->page_rows - 1)))
        return unsupported(e, "page_rows is no power of two from 16 to 1024");
    if (c->num_kv_heads > (1u << 12)) return size_overflow(e, "num_kv_heads");
    if (c->max_sequences > 1024) return size_overflow(e, "max_sequences");
    if (c->page_count >= (1ull << 31)) return size_overflow(e, "page_count");
    if (c->max_table_pages > (1ull << 28)) return size_overflow(e, "max_table_pages");
    if (c->flags) return invalid_argument(e, "flags must be 0");
    uint32_t shift = 0;
    while ((1u << shift) < c->page_rows) ++shift;
    g.kv_heads = uint32_t(c->num_kv_heads);
    g.head_dim = uint32_t(c->head_dim);
    g.page_shift = shift;
    g.ids_at = paged_ids_at(c->max_sequences);
    g.head_stride = c->page_rows * c->head_dim;
    g.side_stride = g.head_stride * g.kv_heads;
    g.page_stride = 2 * g.side_stride;
    uint64_t all = 0;
    if (g.page_stride >= (1ull << 31)) return size_overflow(e, "a page of one layer");  // (4 GiB)
    if (__builtin_mul_overflow(g.page_stride, c->page_count, &layer_stride) ||
        __builtin_mul_overflow(layer_stride, uint64_t(c->layer_count), &all) || __builtin_mul_overflow(all, uint64_t(2), &bytes) ||
        bytes > (1ull << 62))
        return size_overflow(e, "page storage");
    return ITAK_OK;
}

itak_status check_layer(itak_paged *p, uint64_t layer) {
    return layer < p->cfg.layer_count ? itak_status(ITAK_OK) : invalid_layer(p->err, layer, p->cfg.layer_count);
}

itak_status check_rotation(itak_paged *p, const itak_rotation *r) {
    if (!r) return ITAK_OK;
    if (r->cfg.rotary_dim > p->cfg.head_dim) return shape_mismatch(p->err, "rotary_dim", p->cfg.head_dim, r->cfg.rotary_dim);
    if (r->cfg.device != p->cfg.device) return invalid_argument(p->err, "the rotation is another device's");
    return ITAK_OK;
}

itak_status check_tensor(itak_paged *p, const char *what, const itak_rows *v, uint64_t heads, uint32_t elem, bool written) {
    itak_status st = check_rows(p->err, what, v, p->batch.rows, p->cfg.head_dim, written);
    if (st != ITAK_OK) return st;
    if (heads && v->heads != heads) return shape_mismatch(p->err, what, heads, v->heads);
    if (v->elem != ITAK_ELEM_F32 && v->elem != p->cfg.elem)
        return set_error(p->err, ITAK_UNSUPPORTED, what, v->elem, 0, 0, 0, "unsupported: %s is neither f32 nor of the pages' type", what);
    if (elem != ~0u && v->elem != elem)
        return set_error(p->err, ITAK_INVALID_ARGUMENT, what, v->elem, elem, 0, 0, "invalid argument: %s is of another type than the call's other tensors", what);
    return ITAK_OK;
}

uint16_t *layer_base(const itak_paged *p, uint64_t layer) {
    return reinterpret_cast<uint16_t *>(p->storage) + layer * p->layer_stride;
}

// What the kernels multiply products by: to scores in the log2 domain, with a softcap to the argument of its exponential.
float score_scale(const itak_paged *p, uint32_t elem, float scale, float softcap) {
    const float s = std::isnan(scale) ? 1.0f / std::sqrt(float(p->cfg.head_dim)) : scale;
    const float x = softcap > 0.0f ? s * (2.0f * kPagedLog2e / softcap) : s * kPagedLog2e;
    return p->cfg.elem == ITAK_ELEM_F16 && elem == ITAK_ELEM_F32 ? x / kPagedQueryLift : x;
}

itak_status check_attention(itak_paged *p, uint64_t layer, const itak_rows *q, const itak_rows *out, float scale, float softcap,
                            uint64_t window) {
    itak_status st = check_layer(p, layer);
    if (st == ITAK_OK) st = check_tensor(p, "q", q, 0, ~0u, false);
    if (st == ITAK_OK) st = check_tensor(p, "out", out, q->heads, q->elem, true);
    if (st != ITAK_OK) return st;
    if (p->batch.rows && q->data == out->data) return invalid_argument(p->err, "out shares its memory with q");
    if (q->heads % p->cfg.num_kv_heads) return non_divisible(p->err, q->heads, p->cfg.num_kv_heads);
    if (q->heads / p->cfg.num_kv_heads > 64) return unsupported(p->err, "more than 64 query heads a KV head");
    if (q->heads > 65535) return unsupported(p->err, "more than 65535 query heads");
    if (window && window < p->batch.tree_most)
        return set_error(p->err, ITAK_UNSUPPORTED, "window", p->batch.tree_most, window, 0, 0,
                         "unsupported: a window of %llu over a tree of %u rows", ULL(window), p->batch.tree_most);
    if (std::isinf(scale)) return invalid_argument(p->err, "scale is infinite");
    if (!(softcap >= 0.0f) || std::isinf(softcap)) return invalid_argument(p->err, "softcap must be finite and >= 0");
    if (softcap > 0.0f) {
        const float cap_scale = score_scale(p, q->elem, scale, softcap);
        if (!std::isfinite(cap_scale)) return unsupported(p->err, "a softcap so small that scale / softcap is infinite");
        // (Of smaller caps such a scale makes the scores zero.)
        if (softcap > 0x1p24f && cap_scale != 0.0f && std::fabs(cap_scale) < FLT_MIN)
            return unsupported(p->err, "a softcap so large that scale / softcap is none of f32's normal numbers");
        if (std::isinf(softcap * kPagedLog2e)) return unsupported(p->err, "a softcap beyond 2e38");
    }
    return ITAK_OK;
}

// Blocks of all units of a launch: the kernels add them up in 32 bits, rounded up by at most as many again.
constexpr uint64_t kMostBlocks = 1ull << 30;

uint32_t shift_of(uint32_t power) { return uint32_t(__builtin_ctz(power)); }

// How a batch whose rows may be trees is cut: by which kernel, the vectors of a tile, and the blocks of a workgroup's part. The cost of a choice is
// worked out in clocks: of a workgroup what it takes before its first products and behind its last, its steps, or its blocks on their way from L2
// where that is more, and its partial's way out; of the launch its rounds and, where units are split, the join and the partials' way there and back.
// Measured, tiles of 64 and of 128 vectors of the kernel of trees and of 256 of the other, each at its best share: 16 rows at 4,096 17.3, 22.0 and 19.6 us;
// 64 rows at 8,192 42, 29.5 and 40; 4 of 61 in a window of 2,048 27.4, 28.2 and 27.2; 16 of 26 at 8,000 108, 95 and 80; 8 of 32 at 600 17.1, 21.6 and 22.9;
// 64 of 8 at 3,000 72, - and 97; 2 of 256 at 1,000 25, 30 and 34; 20 rows at 60,000 75, 67 and 45.
using TreesCut = PagedBatch::Cut;
TreesCut trees_plan(const PagedBatch &batch, const PagedAttn &a, uint32_t waves, uint32_t chunk_waves, bool f32, uint32_t dp, uint32_t cus) {
    struct Run {
        uint32_t vectors, blocks;
    };
    std::vector<Run> runs;
    uint32_t longest = 1, widest = 1;
    for (uint32_t i = 0; i < a.items; ++i) {
        const uint32_t *it = batch.head.data() + kPagedItem0 + 4 * i;
        const uint64_t vectors = uint64_t(it[1]) * a.group;
        if (vectors < a.v_from || vectors > a.v_to) continue;
        const uint32_t blocks = (it[0] + it[1] + 31) / 32 - paged_first_block(it[0], a.window);
        runs.push_back({uint32_t(vectors), blocks});
        longest = std::max(longest, blocks), widest = std::max(widest, uint32_t(vectors));
    }
    TreesCut best{0, chunk_waves != 0, 32 * (chunk_waves ? chunk_waves : waves), longest};
    double lowest = 1e300;
    auto look = [&](bool chunk, uint32_t sets, uint32_t groups) {
        const uint32_t tile = 32 * sets;
        // Clocks of a step, of 128 channels: chunks' wavefronts work at their products and their softmax at once, four groups send twice the loads of two, and
        // tensors of f32 are several products each (of chunks, whose tiles are half as large then, about as much in all).
        const double step = (chunk ? 1900.0 : (groups > 2 ? 3300.0 : 2450.0) * (f32 ? 2.2 : 1.0) * (waves == 8 ? 1.0 : 0.6)) * dp / 128;
        for (uint32_t share = longest;;) {
            uint64_t parts = 0, work = 0, once = 0;
            for (const Run &r : runs) {
                const uint64_t tiles = (r.vectors + tile - 1) / tile;
                parts += tiles * ((r.blocks + share - 1) / share), work += tiles * r.blocks, once += r.blocks;
            }
            parts *= a.g.kv_heads, work *= a.g.kv_heads, once *= a.g.kv_heads;
            if (parts > kPagedTreesGroups && share != longest) break;
            const bool split = share < longest;
            // A block's way: of what no other tile reads at 6.2 TB/s among all.
            const double load = std::max(280.0, 1420.0 * once / work * std::min(1.0, double(parts) / cus)) * dp / 128;
            auto time = [&](double blocks) { return std::max(std::ceil(blocks / groups) * step, blocks * load); };
            const double beside = chunk ? 13000.0 : 11000.0 + (groups > 1 ? 2000.0 : 1000.0), partial = split ? tile * dp / 16.0 : 0.0;
            const double alone = time(share) + beside + partial;
            const double among = double(parts) / cus * (time(double(work) / parts) + beside + partial) + time(share) / 2;
            const double cost = (parts <= cus ? alone : std::max(alone, among)) + (split ? 8000.0 + parts * tile * dp / 500.0 : 0.0);
            if (cost < lowest) lowest = cost, best = {0, chunk, tile, share};
            if (share <= 2 || parts > 2 * cus) break;
            // (Shares that are whole steps of the groups.)
            share = std::max<uint32_t>(2, std::min((share - 1) / groups * groups, share * 7 / 8 / groups * groups));
        }
    };
    // (Tiles of one set, each read by itself, were behind those of two: 4 of 16 rows by 4 heads at 1,000 18.4 us and 16.2.)
    for (uint32_t sets = 2; sets <= waves; sets *= 2) {
        if (16 * sets >= widest && sets > 2) break;
        look(false, sets, waves / sets);
    }
    if (chunk_waves) look(true, chunk_waves, 1);
    return best;
}

// Units and blocks of the items a launch takes, how their line is cut, and where in it inline items begin; `whole`: no unit is split.
itak_status count_units(itak_paged *p, PagedAttn &a, uint64_t &work, bool &whole, bool known = false) {
    uint32_t longest = 0;
    auto each = [&](uint32_t pad, auto item) {
        uint64_t at = 0, units = 0;
        for (uint32_t i = 0; i < a.items; ++i) {
            const uint32_t *it = p->batch.head.data() + kPagedItem0 + 4 * i;
            const uint64_t vectors = uint64_t(it[1]) * a.group;
            item(i, at, units);
            if (vectors < a.v_from || vectors > a.v_to) continue;
            const uint64_t tiles = (vectors + a.tile - 1) / a.tile * (a.apart ? 1 : a.g.kv_heads);
            const uint32_t blocks = (it[0] + it[1] + 31) / 32 - paged_first_block(it[0], a.window);
            units += tiles;
            at += tiles * paged_run(blocks, pad);
            longest = std::max(longest, blocks);
        }
        item(a.items, at, units);
    };
    uint64_t units = 0;
    each(0, [&](uint32_t, uint64_t at, uint64_t u) { work = at, units = u; });
    // (Of the kernel of many rows a unit is a workgroup of up to 512 threads, and a launch's threads are counted in 32 bits; where units are
    // dealt to parts they are few.)
    if (work >= kMostBlocks || units > (1ull << 32) / 512 - 1) return size_overflow(p->err, "blocks of the batch's attention");
    a.units = uint32_t(units);
    if (a.apart) {
        const uint32_t room = std::max(1u, kPagedTreesGroups / a.g.kv_heads), share = a.share;
        // (Where the batch is not known as many workgroups as the cut takes here, and one for every compute unit: for other lengths.)
        const uint64_t parts = units + (share < longest ? (work + share - 1) / share : 0);
        const uint64_t asked = known ? room : std::max<uint64_t>(parts, std::max(1u, compute_units()) / a.g.kv_heads);
        a.groups = std::max(a.units, uint32_t(std::min<uint64_t>(room, asked)));
        whole = a.groups == a.units;
        if (whole) a.least = ~0u;
        if (known) {
            a.share = a.pad = share;
            for (uint32_t i = 0; i < kPagedInline; ++i) a.start[i] = a.unit0[i] = ~0u;
            uint64_t total = 0;
            each(share, [&](uint32_t i, uint64_t at, uint64_t u) {
                if (i < a.inline_items) a.start[i] = uint32_t(at), a.unit0[i] = uint32_t(u);
                total = at;
            });
            // (Every unit's run is rounded up by less than a share: what the device counts in 32 bits may then be too much.)
            if (total >= 2 * kMostBlocks) return size_overflow(p->err, "blocks of the batch's attention");
            a.total = uint32_t(total);
            whole = share >= longest;
        } else {
            a.share = 0;
        }
        // (Workgroups that would find nothing are left out where the batch is known.)
        a.across = known ? a.total / share : a.groups;
        return ITAK_OK;
    }
    // (The kernel of many rows has no line.)
    const PagedCut cut = a.parts ? PagedCut{} : paged_cut(uint32_t(work), a.units, longest, a.groups, a.least);
    whole = cut.pad >= longest;
    if (!known) return ITAK_OK;
    a.share = cut.share, a.pad = cut.pad;
    for (uint32_t i = 0; i < kPagedInline; ++i) a.start[i] = a.unit0[i] = ~0u;
    each(cut.pad, [&](uint32_t i, uint64_t at, uint64_t u) {
        if (i < a.inline_items) a.start[i] = uint32_t(at), a.unit0[i] = uint32_t(u);
        a.total = uint32_t(at);
    });
    return ITAK_OK;
}

// What a call's attention launches: found out, and its memory had, before the call enqueues anything.
struct AttnPlan {
    PagedAttn few{}, trees{}, many{};
    uint32_t sets = 0;       // of the kernel of few rows; 0: it has no items
    bool merge_few = false;
    bool has_trees = false, join_trees = false, trees_as_many = false;
    bool has_many = false;
};

// Vectors' places in the partials of the kernel of trees: as many as any call of it takes, which one has from itak_paged_enable_trees on. (A captured one may be
// planned for other lengths than the calls before it.)
uint64_t trees_places(const PagedGeom &g) { return (uint64_t(kPagedTreesGroups) + g.kv_heads) * 256; }

// The partials of all launches lie in one place: they run one after the other.
itak_status workspace(itak_paged *p, AttnPlan &plan, uint32_t dp) {
    auto slots = [](const PagedAttn &a) { return a.parts ? (a.parts > 1 ? uint64_t(a.units) * a.parts : 0) : uint64_t(a.groups) + a.units; };
    auto vectors = [&](const PagedAttn &a) { return a.apart ? trees_places(a.g) : slots(a) * a.tile; };
    auto sums = [&](const PagedAttn &a) { return vectors(a) * dp * sizeof(float); };
    uint64_t need = 0;
    for (const PagedAttn *a : {&plan.few, &plan.trees, &plan.many}) need = std::max(need, sums(*a) + vectors(*a) * sizeof(float2));
    void *ws = p->ws;
    const itak_status st = grow(p, &ws, &p->ws_bytes, need, "split workspace");
    p->ws = static_cast<float *>(ws);
    for (PagedAttn *a : {&plan.few, &plan.trees, &plan.many}) {
        a->ws_acc = p->ws;
        a->ws_ml = reinterpret_cast<float2 *>(reinterpret_cast<unsigned char *>(p->ws) + sums(*a));
    }
    return st;
}

// Parts of a unit's keys in the kernel of many rows: as many as fill the device, each part a workgroup that costs some blocks'
// time beside its own, and more where the merge has more than 64 of them to join (64 vectors over 20,000 16.7 us with 64 parts and 20.2
// with 256, over 100,000, two of them, 44.3 with 64 and 34.1 with 128).
uint32_t chunk_parts(uint32_t units, uint64_t work, uint32_t places) {
    const double blocks = double(work) / units;
    uint32_t best = 1;
    double least = 1e300;
    for (uint32_t s = 1; s <= 256 && s <= blocks / 2 + 1; ++s) {
        const double extra = s > 64 ? 24.0 : s > 1 ? 8.0 : 0.0;
        const double rounds = std::ceil(double(units) * s / places), cost = rounds * (std::ceil(blocks / s) + extra);
        if (cost < least * 0.97) least = cost, best = s;
        if (units * s > 2 * places) break;
    }
    return best;
}

// q is as it attends: turned where it has to be.
itak_status plan_attention(itak_paged *p, uint64_t layer, const itak_rows &q, const itak_rows &out, float scale, float softcap,
                           uint64_t window, AttnPlan &plan) {
    // (A call that is being captured is replayed over other batches.)
    const bool captured = capturing(p->stream);
    const uint32_t d = uint32_t(p->cfg.head_dim);
    const uint32_t group = uint32_t(q.heads / p->cfg.num_kv_heads);
    PagedAttn &a = plan.few;
    a.g = p->g;
    a.batch = p->batch_dev;
    a.layer_base = layer_base(p, layer);
    a.q = rows_view(q, d);
    a.out = rows_view(out, d);
    a.rows = p->batch.rows;
    a.items = p->batch.items;
    a.group = group;
    a.group_magic = group > 1 ? uint32_t((1ull << 32) / group + ((1ull << 32) % group != 0)) : 0;
    if (uint64_t(a.rows) * group >= (1ull << 26)) return size_overflow(p->err, "query vectors of the batch");
    // A handle that takes trees captures launches that find out whether the batch has them.
    if (p->batch.trees || (captured && p->tree_dev)) a.tree = p->tree_dev;
    const bool known = !captured && !p->batch.on_device;
    if (a.items <= kPagedInline && known) {
        a.inline_items = a.items;
        for (PagedItemWords &w : a.item) w.row0 = ~0u;
        std::memcpy(a.item, p->batch.head.data() + kPagedItem0, a.items * sizeof(PagedItemWords));
    }
    a.q_on_16 = rows_on_16(q, d);
    a.out_on_16 = rows_on_16(out, d);
    a.scale_log2 = score_scale(p, q.elem, scale, softcap);
    a.cap_log2 = softcap * kPagedLog2e;
    a.window = uint32_t(std::min<uint64_t>(window, 1ull << 31));
    a.zeros = p->batch_dev + p->zeros_at;
    const uint32_t dp = paged_padded(d), cus = std::max(1u, compute_units());
    // Items of few query vectors a KV head and items of many are launches of their own: a prompt's chunk among other
    // sequences' tokens is common. Up to 32 vectors are few (4 of 4 rows by 8 heads at 8,192 in f32 22.0 us there and 25.5 in the
    // kernel of many, 16 in f16 59.3 and 66.5); of 56 the kernel of many is level (4 at 8,192 in f16 25.9 and 25.5) or ahead (in f32 32.7
    // and 27.8, 64 at 600 47.7 and 26.7), though tiles of four sets of 16 had been made for them.
    const uint32_t few_most = 2 * kPagedSet;
    const bool chunks = paged_chunk_takes(dp, p->cfg.elem, q.elem);
    // Of a batch whose rows may be trees those of more than few vectors are one launch, of the kernel of trees or of that of many rows.
    uint32_t most_few = 0;
    bool many = false;
    for (uint32_t i = 0; i < a.items; ++i) {
        const uint64_t vectors = uint64_t(p->batch.head[kPagedItem0 + 4 * i + 1]) * group;
        if (a.tree && vectors > few_most)
            plan.has_trees = true;
        else if (chunks && vectors > few_most)
            many = true;
        else
            most_few = std::max(most_few, uint32_t(std::min<uint64_t>(vectors, few_most)));
    }
    bool whole = false;
    uint64_t work = 0;
    if (many) {
        PagedAttn &b = plan.many = a;
        plan.has_many = true;
        b.tile = 32 * paged_chunk_waves(dp, q.elem);
        b.tile_shift = shift_of(b.tile);
        b.v_from = few_most + 1, b.v_to = ~0u;
        b.parts = 1;
        const itak_status st = count_units(p, b, work, whole, known);
        if (st != ITAK_OK) return st;
        b.parts = chunk_parts(b.units, work, cus * kPagedChunkGroupsPerCu);
    }
    if (plan.has_trees) {
        PagedAttn &b = plan.trees = a;
        b.v_from = few_most + 1, b.v_to = ~0u;
        b.apart = 1;
        // (Once a batch: a layer after another asks the same, and over 256 items the answer takes some tens of microseconds.)
        TreesCut &cut = p->batch.cuts[a.window ? 1 : 0];
        const uint64_t key = (uint64_t(q.heads) * 2 + (q.elem == ITAK_ELEM_F32)) << 32 | (a.window ? a.window : 1);
        if (cut.key != key) {
            cut = trees_plan(p->batch, b, paged_trees_waves(dp, p->cfg.elem, q.elem), chunks ? paged_chunk_waves(dp, q.elem) : 0,
                             q.elem == ITAK_ELEM_F32, dp, cus);
            cut.key = key;
        }
        b.tile = cut.tile, b.share = cut.share;
        plan.trees_as_many = cut.chunk;
        b.tile_shift = shift_of(b.tile);
        b.least = std::max(2u, cut.chunk ? 2u : paged_trees_waves(dp, p->cfg.elem, q.elem) * 32 / cut.tile);  // (a step's blocks)
        const itak_status st = count_units(p, b, work, whole, known);
        if (st != ITAK_OK) return st;
        plan.join_trees = !whole;
    }
    if (most_few) {
        plan.sets = most_few <= kPagedSet ? 1 : 2;
        a.tile = plan.sets * kPagedSet;
        a.tile_shift = shift_of(a.tile);
        a.v_from = 1, a.v_to = chunks || a.tree ? few_most : ~0u;
        a.groups = std::min(cus * paged_few_groups_per_cu(dp, p->cfg.elem, q.elem, plan.sets, a.tree != nullptr), kPagedMostParts);
        a.least = 4;
        a.parts = 0;
        const itak_status st = count_units(p, a, work, whole, known);
        if (st != ITAK_OK) return st;
        plan.merge_few = !known || !whole;
    }
    if (const auto &c = p->captured_batch; captured && c.rows && !(p->batch.capture && p->batch.capture == capture_of(p->stream))) {
        // (Of batches that other graphs set the same as of those that are set from now on: paged_replays_hold.)
        const uint64_t units = std::max({plan.few.units, plan.trees.units, plan.many.units});
        if (units * ((c.position + c.rows + 31) / 32 - paged_first_block(c.position, a.window)) >= kMostBlocks)
            return size_overflow(p->err, "attention over a captured batch");
        if (a.window && a.window < c.tree_most)
            return set_error(p->err, ITAK_UNSUPPORTED, "window", c.tree_most, a.window, 0, 0,
                             "unsupported: a window of %u over a tree of %u rows (of a batch that was captured)", a.window, c.tree_most);
    }
    const itak_status st = workspace(p, plan, dp);
    // (A graph looks at all items of the batch that is there when it runs. Sequences without rows are left out of one set here, and count among those of a
    // handle that takes trees and of a batch that the device makes.)
    if (captured)
        for (PagedAttn *b : {&plan.few, &plan.trees, &plan.many}) b->items = p->cfg.max_sequences;
    if (st == ITAK_OK && captured) {
        itak_paged::Captured &c = p->captured[a.window ? 1 : 0];
        c.units = std::max<uint64_t>({c.units, plan.few.units, plan.trees.units, plan.many.units});
        c.window = std::max(c.window, a.window);
        if (a.window && p->tree_dev) c.least_window = c.least_window ? std::min(c.least_window, a.window) : a.window;
    }
    return st;
}

}  // namespace

// Whether the captured calls' replays over a batch (of as many units) can count their blocks, and whether its trees fit their windows.
itak_status itak::paged_replays_hold(const itak_paged *p, const PagedBatch &batch) {
    const std::vector<uint32_t> &head = batch.head;
    for (const itak_paged::Captured &c : p->captured) {
        for (size_t at = kPagedItem0; c.units && at < head.size(); at += 4) {
            const uint32_t blocks = (head[at] + head[at + 1] + 31) / 32 - paged_first_block(head[at], c.window);
            if (c.units * blocks >= kMostBlocks) return size_overflow(p->err, "a captured attention over the batch");
        }
        if (c.least_window && batch.tree_most > c.least_window)
            return set_error(p->err, ITAK_UNSUPPORTED, "window", batch.tree_most, c.least_window, 0, 0,
                             "unsupported: a window of %u over a tree of %u rows (an attention that was captured has it)", c.least_window, batch.tree_most);
    }
    return ITAK_OK;
}

itak_status itak::paged_reserve_trees(itak_paged *p) {
    void *ws = p->ws;
    const uint64_t bytes = trees_places(p->g) * (paged_padded(p->g.head_dim) * sizeof(float) + sizeof(float2));
    const itak_status st = grow(p, &ws, &p->ws_bytes, bytes, "allocate the partials of trees", true);
    p->ws = static_cast<float *>(ws);
    return st;
}

namespace {

itak_status run_attention(itak_paged *p, uint32_t elem, const AttnPlan &plan) {
    const bool trees = plan.few.tree != nullptr;
    if (plan.sets) {
        const hipError_t he =
            p->cfg.elem == ITAK_ELEM_F16
                ? (elem == ITAK_ELEM_F32 ? (trees ? launch_paged_few_tree_f16_f32 : launch_paged_few_f16_f32)
                                           : (trees ? launch_paged_few_tree_f16 : launch_paged_few_f16))(plan.sets, plan.few, p->stream)
                : (elem == ITAK_ELEM_F32 ? (trees ? launch_paged_few_tree_bf16_f32 : launch_paged_few_bf16_f32)
                                         : (trees ? launch_paged_few_tree_bf16 : launch_paged_few_bf16))(plan.sets, plan.few, p->stream);
        HIP_TRY(p, he, "launch paged attention of few rows");
        if (plan.merge_few)
            HIP_TRY(p, (trees ? launch_paged_few_join : launch_paged_merge)(elem, plan.few, p->stream), "launch the merge of paged attention");
    }
    if (plan.has_trees) {
        const bool f16 = p->cfg.elem == ITAK_ELEM_F16, f32 = elem == ITAK_ELEM_F32;
        const auto launch = plan.trees_as_many ? (f16 ? (f32 ? launch_paged_chunk_tree_f16_f32 : launch_paged_chunk_tree_f16)
                                                      : (f32 ? launch_paged_chunk_tree_bf16_f32 : launch_paged_chunk_tree_bf16))
                                               : (f16 ? (f32 ? launch_paged_trees_f16_f32 : launch_paged_trees_f16)
                                                      : (f32 ? launch_paged_trees_bf16_f32 : launch_paged_trees_bf16));
        const hipError_t he = launch(plan.trees, p->stream);
        HIP_TRY(p, he, "launch paged attention of trees");
        if (plan.join_trees) HIP_TRY(p, launch_paged_join(elem, plan.trees, p->stream), "launch the join of paged attention");
    }
    if (plan.has_many) {
        const hipError_t he = p->cfg.elem == ITAK_ELEM_F16
                                  ? (elem == ITAK_ELEM_F32 ? launch_paged_chunk_f16_f32 : launch_paged_chunk_f16)(plan.many, p->stream)
                                  : (elem == ITAK_ELEM_F32 ? launch_paged_chunk_bf16_f32 : launch_paged_chunk_bf16)(plan.many, p->stream);
        HIP_TRY(p, he, "launch paged attention of many rows");
        if (plan.many.parts > 1) HIP_TRY(p, launch_paged_merge(elem, plan.many, p->stream), "launch the merge of paged attention");
    }
    return ITAK_OK;
}

itak_status run_append(itak_paged *p, uint64_t layer, const itak_rows &k, const itak_rows &v, const itak_rotation *rotation,
                       const itak_rows *q, const itak_rows *q_out) {
    const uint32_t d = uint32_t(p->cfg.head_dim);
    PagedAppend a{};
    a.g = p->g;
    a.batch = p->batch_dev;
    a.tree = p->tree_dev;
    a.layer_base = layer_base(p, layer);
    a.k = rows_view(k, d);
    a.v = rows_view(v, d);
    a.r = rotation_view(rotation);
    bool by_8 = pieces_of_8(d, a.r.half, a.r.interleaved) && rows_on_16(k, d) && rows_on_16(v, d);
    if (q) {
        a.q = rows_view(*q, d);
        a.q_out = rows_view(*q_out, d);
        a.q_heads = q->heads;
        by_8 = by_8 && rows_on_16(*q, d) && rows_on_16(*q_out, d);
    }
    HIP_TRY(p, launch_paged_append(p->cfg.elem, k.elem, by_8, a, p->batch.rows, p->stream), "launch the append to pages");
    return ITAK_OK;
}

// Queries alone, turned by the batch's positions.
itak_status run_append_queries(itak_paged *p, const itak_rows &q, const itak_rows &q_out, const itak_rotation *rotation) {
    const uint32_t d = uint32_t(p->cfg.head_dim);
    PagedAppend a{};
    a.g = p->g;
    a.g.kv_heads = 0;
    a.batch = p->batch_dev;
    a.tree = p->tree_dev;
    a.r = rotation_view(rotation);
    a.q = rows_view(q, d);
    a.q_out = rows_view(q_out, d);
    a.q_heads = q.heads;
    const bool by_8 = pieces_of_8(d, a.r.half, a.r.interleaved) && rows_on_16(q, d) && rows_on_16(q_out, d);
    HIP_TRY(p, launch_paged_append(p->cfg.elem, q.elem, by_8, a, p->batch.rows, p->stream), "launch a rotation of queries");
    return ITAK_OK;
}

// A dense buffer for q's rows, turned.
itak_status turned_rows(itak_paged *p, const itak_rows &q, itak_rows &out) {
    const uint64_t bytes = uint64_t(p->batch.rows) * q.heads * p->cfg.head_dim * elem_size(q.elem);
    itak_status st = grow(p, &p->turned, &p->turned_bytes, bytes, "rotated queries");
    out = itak_rows{p->turned, q.elem, q.heads, 0, 0};
    return st;
}

// Whether the parents of a batch's new rows make trees; the largest tree's rows.
itak_status check_trees(itak_paged *p, const itak_paged_item *items, uint32_t count, const int32_t *parents, uint32_t rows, uint32_t &most) {
    if (!p->tree_dev) return unsupported(p->err, "a batch of trees of a paged cache that takes none (itak_paged_enable_trees)");
    if (rows > p->tree_rows)
        return set_error(p->err, ITAK_CAPACITY_EXCEEDED, "rows of trees", rows, p->tree_rows, 0, 0,
                         "a batch of trees of %u rows, the paged cache takes %llu", rows, ULL(p->tree_rows));
    most = 0;
    for (uint32_t i = 0; i < count; parents += items[i].rows, ++i) {
        const uint64_t n = items[i].rows, wrong = tree_first_wrong(parents, n);
        if (wrong < n)
            return set_error(p->err, ITAK_INVALID_ARGUMENT, "parents", i, wrong, 0, 0,
                             "invalid argument: item %u: the parent of row %llu is %d, no row before it and not -1", i, ULL(wrong),
                             int(parents[wrong]));
        if (tree_is_chain(parents, n)) continue;
        if (n > kTreeRows)
            return set_error(p->err, ITAK_UNSUPPORTED, "rows of a tree", i, n, 0, 0,
                             "unsupported: item %u: a tree of %llu rows, of more than %u only chains are taken", i, ULL(n), kTreeRows);
        most = std::max(most, uint32_t(n));
    }
    return ITAK_OK;
}

itak_status set_batch(itak_paged *p, const itak_paged_item *items, uint32_t count, const uint32_t *pages, uint64_t page_ids,
                      const int32_t *parents) {
    if (capturing(p->stream)) return invalid_argument(p->err, "the batch is set while the stream is being captured");
    PagedBatch &next = p->next;
    const PagedRefusal r = make_paged_batch(p->limits, items, count, pages, page_ids, p->marks, p->stamp, next, p->tree_dev != nullptr);
    if (r.code != ITAK_OK) return set_error(p->err, r.code, r.what, r.a, r.b, 0, 0, "%s", r.text.c_str());
    next.trees = parents != nullptr, next.on_device = false, next.tree_most = 0, next.capture = 0;
    next.cuts[0] = next.cuts[1] = {};
    if (parents) {
        const itak_status st = check_trees(p, items, count, parents, next.rows, next.tree_most);
        if (st != ITAK_OK) return st;
        next.head[2] = 1;
    }
    if (const itak_status st = paged_replays_hold(p, next); st != ITAK_OK) return st;
    const DeviceScope scope(p->cfg.device);
    HIP_TRY(p, scope.status(), "set the device");
    // The items go up every time, page ids where they are not what the device has: of a sequence that grows, one every
    // page_rows tokens.
    const std::vector<uint32_t> &head = next.head, &ids = next.ids;
    const uint32_t ids_at = p->g.ids_at;
    uint32_t lo = 0, hi = uint32_t(ids.size());
    if (!p->ids_known || p->ids_never_known) std::fill(p->ids_there.begin(), p->ids_there.end(), ~0u);
    p->ids_known = true;
    while (lo < hi && p->ids_there[lo] == ids[lo]) ++lo;
    while (hi > lo && p->ids_there[hi - 1] == ids[hi - 1]) --hi;
    // What the device has is unknown from the first launch to the last.
    std::copy(ids.begin() + lo, ids.begin() + hi, p->ids_there.begin() + lo);
    const bool sent = parents && next.rows && send_tree_batch(p->batch_dev, p->tree_dev, head, ids_at + lo, ids.data() + lo, hi - lo, parents,
                                                              next.rows, next.items, p->stream);
    if (sent) lo = hi;
    for (uint32_t at = 0; !sent && at < head.size();) {
        const uint32_t n = std::min<uint32_t>(uint32_t(head.size()) - at, kManyWords);
        const uint32_t room = at + n == head.size() ? kManyWords - n : 0;
        const uint32_t m = std::min(room, hi - lo);
        send_words(p->batch_dev, at, head.data() + at, n, ids_at + lo, ids.data() + lo, m, p->stream);
        at += n, lo += m;
    }
    for (; lo < hi;) {
        const uint32_t n = std::min(hi - lo, kManyWords);
        send_words(p->batch_dev, ids_at + lo, ids.data() + lo, n, 0, nullptr, 0, p->stream);
        lo += n;
    }
    hipError_t he = hipSuccess;
    if (parents && next.rows && !sent) {
        uint32_t *const there = p->tree_dev + p->tree_rows * kTreeStride;
        const uint32_t *words = reinterpret_cast<const uint32_t *>(parents);
        for (uint32_t at = 0; at < next.rows; at += kManyWords)
            send_words(there, at, words + at, std::min(next.rows - at, kManyWords), 0, nullptr, 0, p->stream);
        he = launch_paged_records(p->batch_dev, next.items, reinterpret_cast<const int32_t *>(there), p->tree_dev, p->stream);
    }
    if (he == hipSuccess) he = hipGetLastError();
    if (he != hipSuccess) {
        std::fill(p->ids_there.begin(), p->ids_there.end(), ~0u);
        p->batch = PagedBatch{};
        return hip_error(p->err, he, "send a batch to the device");
    }
    std::swap(p->batch, p->next);
    return ITAK_OK;
}

}  // namespace

extern "C" {

uint64_t itak_paged_storage_bytes(const itak_paged_config *config) {
    PagedGeom g{};
    uint64_t stride = 0, bytes = 0;
    ErrorState e;
    return check_config(e, config, g, stride, bytes) == ITAK_OK ? bytes : 0;
}

itak_status itak_paged_create(const itak_paged_config *config, itak_paged **out) {
    ErrorState &e = thread_error();
    if (!out) return invalid_argument(e, "out is null");
    *out = nullptr;
    PagedGeom g{};
    uint64_t stride = 0, bytes = 0;
    if (itak_status st = check_config(e, config, g, stride, bytes); st != ITAK_OK) return st;
    if (config->storage) {
        if (config->storage_bytes < bytes) return shape_mismatch(e, "storage_bytes", bytes, config->storage_bytes);
        if (reinterpret_cast<uintptr_t>(config->storage) % 16) return invalid_argument(e, "storage does not start on 16 bytes");
    }
    itak_paged *p = nullptr;
    hipError_t he = hipSuccess;
    try {
        p = new itak_paged;
        p->cfg = *config;
        if (p->cfg.max_table_pages == 0) p->cfg.max_table_pages = std::min<uint64_t>(config->page_count, 1ull << 28);
        p->g = g;
        p->layer_stride = stride;
        p->bytes = bytes;
        p->limits = PagedLimits{config->page_count, config->page_rows, config->max_sequences, p->cfg.max_table_pages};
        p->marks.assign(config->page_count, 0);
        p->ids_there.assign(p->cfg.max_table_pages, 0);
        p->batch.head.assign(kPagedItem0, 0);
    } catch (const std::bad_alloc &) {
        delete p;
        return invalid_argument(e, "out of host memory");
    }
    const DeviceScope scope(config->device);
    he = scope.status();
    p->zeros_at = (p->g.ids_at + p->cfg.max_table_pages + 3) / 4 * 4;
    const uint64_t words = (p->zeros_at + 4 + 2 * uint64_t(config->max_sequences)) * sizeof(uint32_t);
    if (he == hipSuccess) he = hipMalloc(reinterpret_cast<void **>(&p->batch_dev), words);
    if (he == hipSuccess) he = hipMemset(p->batch_dev, 0, words);  // (an empty batch)
    if (he == hipSuccess) p->rows_dev = p->batch_dev + p->zeros_at + 4;
    p->storage = static_cast<unsigned char *>(config->storage);
    p->owns = !config->storage;
    if (he == hipSuccess && p->owns) {
        he = hipMalloc(reinterpret_cast<void **>(&p->storage), bytes);
        if (he == hipSuccess) he = hipMemset(p->storage, 0, bytes);
    }
    if (he == hipSuccess) he = hipDeviceSynchronize();  // (whatever stream comes first finds both)
    if (he != hipSuccess) {
        (void)hipGetLastError();
        if (p->batch_dev) (void)hipFree(p->batch_dev);
        if (p->owns && p->storage) (void)hipFree(p->storage);
        delete p;
        return hip_error(e, he, "allocate a paged cache");
    }
    ITAK_DIAG("paged cache built layers=%u kv_heads=%llu head_dim=%llu elem=%s pages=%llu page_rows=%u bytes=%llu", config->layer_count,
              ULL(config->num_kv_heads), ULL(config->head_dim), config->elem == ITAK_ELEM_F16 ? "f16" : "bf16",
              ULL(config->page_count), config->page_rows, ULL(bytes));
    *out = p;
    return ITAK_OK;
}

void itak_paged_destroy(itak_paged *paged) {
    if (!paged) return;
    const DeviceScope scope(paged->cfg.device);
    (void)hipStreamSynchronize(paged->stream);
    if (paged->batch_dev) (void)hipFree(paged->batch_dev);
    if (paged->tree_dev) (void)hipFree(paged->tree_dev);
    if (paged->owns && paged->storage) (void)hipFree(paged->storage);
    for (void *b : paged->buffers) (void)hipFree(b);
    delete paged;
}

const char *itak_paged_last_error(const itak_paged *paged) {
    return paged ? paged->err.message.c_str() : thread_error().message.c_str();
}

itak_status itak_paged_last_error_info(const itak_paged *paged, itak_error_info *out) {
    if (!out) return ITAK_INVALID_ARGUMENT;
    *out = paged ? paged->err.info : thread_error().info;
    return ITAK_OK;
}

itak_status itak_paged_set_stream(itak_paged *paged, void *hip_stream) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    paged->stream = static_cast<hipStream_t>(hip_stream);
    return ITAK_OK;
}

itak_status itak_paged_synchronize(itak_paged *paged) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, hipStreamSynchronize(paged->stream), "synchronize");
    return ITAK_OK;
}

void *itak_paged_storage(const itak_paged *paged) { return paged ? paged->storage : nullptr; }

itak_status itak_paged_set_batch(itak_paged *paged, const itak_paged_item *items, uint32_t count, const uint32_t *pages,
                                 uint64_t page_ids) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    try {
        return set_batch(paged, items, count, pages, page_ids, nullptr);
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
}

itak_status itak_paged_set_batch_tree(itak_paged *paged, const itak_paged_item *items, uint32_t count, const uint32_t *pages,
                                      uint64_t page_ids, const int32_t *parents) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    if (!parents) return invalid_argument(paged->err, "parents are null");
    try {
        return set_batch(paged, items, count, pages, page_ids, parents);
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
}

itak_status itak_paged_append_device(itak_paged *paged, uint64_t layer, const itak_rows *k, const itak_rows *v,
                                     const itak_rotation *rotation) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_layer(paged, layer);
    if (st == ITAK_OK) st = check_tensor(paged, "k", k, paged->cfg.num_kv_heads, ~0u, false);
    if (st == ITAK_OK) st = check_tensor(paged, "v", v, paged->cfg.num_kv_heads, k->elem, false);
    if (st == ITAK_OK) st = check_rotation(paged, rotation);
    if (st != ITAK_OK || paged->batch.rows == 0) return st;
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    return run_append(paged, layer, *k, *v, rotation, nullptr, nullptr);
}

itak_status itak_paged_attention_device(itak_paged *paged, uint64_t layer, const itak_rows *q, const itak_rows *out, float scale,
                                        float softcap, uint64_t window, const itak_rotation *rotation) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_attention(paged, layer, q, out, scale, softcap, window);
    if (st == ITAK_OK) st = check_rotation(paged, rotation);
    if (st != ITAK_OK || paged->batch.rows == 0) return st;
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    try {
        itak_rows turned = *q;
        AttnPlan plan;
        if (rotation) st = turned_rows(paged, *q, turned);
        if (st == ITAK_OK) st = plan_attention(paged, layer, turned, *out, scale, softcap, window, plan);
        if (st == ITAK_OK && rotation) st = run_append_queries(paged, *q, turned, rotation);
        return st == ITAK_OK ? run_attention(paged, q->elem, plan) : st;
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
}

itak_status itak_paged_step_device(itak_paged *paged, uint64_t layer, const itak_rows *q, const itak_rows *k, const itak_rows *v,
                                   const itak_rows *out, float scale, float softcap, uint64_t window,
                                   const itak_rotation *rotation) {
    if (!paged) return ITAK_INVALID_ARGUMENT;
    itak_status st = check_attention(paged, layer, q, out, scale, softcap, window);
    if (st == ITAK_OK) st = check_tensor(paged, "k", k, paged->cfg.num_kv_heads, q->elem, false);
    if (st == ITAK_OK) st = check_tensor(paged, "v", v, paged->cfg.num_kv_heads, q->elem, false);
    if (st == ITAK_OK) st = check_rotation(paged, rotation);
    if (st != ITAK_OK || paged->batch.rows == 0) return st;
    const DeviceScope scope(paged->cfg.device);
    HIP_TRY(paged, scope.status(), "set the device");
    try {
        itak_rows turned = *q;
        AttnPlan plan;
        if (rotation) st = turned_rows(paged, *q, turned);
        if (st == ITAK_OK) st = plan_attention(paged, layer, turned, *out, scale, softcap, window, plan);
        if (st == ITAK_OK) st = run_append(paged, layer, *k, *v, rotation, rotation ? q : nullptr, &turned);
        return st == ITAK_OK ? run_attention(paged, q->elem, plan) : st;
    } catch (const std::bad_alloc &) {
        return invalid_argument(paged->err, "out of host memory");
    }
}

}  // extern "C"
