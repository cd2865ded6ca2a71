// drafts.hip -- drafted tokens and shared blocks (include/maplemoe.h, Part 3): argument checks and launches.
#include "paged_host.h"
#include "drafts.h"
#include "attn_tree.h"

// words: without MMOE_TREE_WINDOW
static int check_bits(const char *who, const mmoe_attn_args *p, const mmoe_kv_cache *kv, int words) {
    if (check_attn(who, p, kv)) return -1;
    if (p->hi) REFUSE("%s: hi is set (new tokens are seen by their bits)", who);
    if (words < 1 || words > MMOE_TREE_MAX / 64) REFUSE("%s: %d words of bits outside 1..%d", who, words, MMOE_TREE_MAX / 64);
    if (p->max_q > 64 * words) REFUSE("%s: max_q %d for %d words of bits", who, p->max_q, words);
    return 0;
}

// How a call of mmoe_attn_tree is divided (attn_tree.h). Only the values in the arguments count (a captured call keeps its grid). The numbers of
// workgroups are for the 256 compute units of the one device that the kernels are built and were measured for.
struct TreePlan {
    int room, most_waves, tiles;
    unsigned wgs, join;
    bool many, deep, fits;
    size_t results, bytes;
};
static TreePlan tree_plan(const mmoe_attn_args &a, const mmoe_kv_cache &kv) {
    TreePlan p = {};
    const int group = a.heads / kv.heads;
    const int64_t rows = (int64_t)a.ntok * group, most = (int64_t)std::min(a.max_q, a.ntok) * group;
    // sequences with tokens; row tiles of their own (and waves of 32 rows), all row tiles
    const int64_t busy = std::min(a.nseq, a.ntok), own = std::min(busy * ((most + ATT_BM - 1) / ATT_BM), rows / ATT_BM + busy), own_waves = std::min(busy * ((most + 31) / 32), rows / 32 + busy);
    const int64_t sh_tiles = a.shared ? (rows + ATT_BM - 1) / ATT_BM : 0, tiles = own + sh_tiles;
    // Row tiles of so few positions, and so many of them, that they stay whole: nothing to join (32 drafts of 64 tokens in a window of 512, 256 row tiles:
    // 25 us, cut 36; 24 drafts, 192: 23.6, cut 29.2; 48 drafts of 4 over 600, 192: 18.9, cut 22.3)
    const int64_t most_steps = (a.window ? std::min<int64_t>(a.max_len, (int64_t)a.window + a.max_q + TREE_BN) : a.max_len) / TREE_BN + 1;
    const bool whole = !a.shared && most_steps <= 12 && tiles * kv.heads >= 192;
    // What the card holds at once: two workgroups per compute unit, three with heads of 64 (64 drafts of 10 to 40 tokens over 50 to 3000 positions, heads of 128:
    // 68 us, with 768 pieces 75; 17 drafts behind 2048 shared positions, heads of 64: 32 us, with 512 pieces 37, but 16 of 20 over 3000 23.4, with 512 21.9)
    const int once = kv.head_dim == 64 ? 768 : 512;
    const int room = std::max(1, once / kv.heads);
    p.room = whole ? 0 : room;
    const int64_t most_pieces = std::max(tiles <= room ? (int64_t)room : room + tiles, tiles), pieces = whole ? tiles : most_pieces, join = own * kv.heads * 4;
    // Few row tiles, so perhaps many results of each, and few workgroups of 32 rows and a key/value head: eight workgroups for one (26 tokens over 700
    // positions, 16: 12.5 us instead of 14.6; over 30000 34 instead of 66; 3 drafts of 60 over 3000, 96: 24.7 instead of 26; 16 of 20 over 2000, 256: 28.6 instead of 27.5)
    p.deep = join < 128;
    p.many = a.nseq > 64;
    // Of up to 64 sequences a workgroup for each piece that there may be. Of more a workgroup for each that the card holds at once: 64 drafts of 20 tokens in
    // a batch of 1024 (4096) sequences, the others without, 54 (73) us instead of 76 (374); 256 drafts of 4 over 1500, all there, 154 instead of 149
    const int64_t wgs = std::min((pieces * kv.heads + 7) & ~(int64_t)7, p.many ? (int64_t)once : INT64_MAX);
    p.fits = tiles * ((int64_t)a.max_len / TREE_BN + 2) <= INT32_MAX && std::max(wgs, join * (p.deep ? 8 : 1)) * 256 <= (int64_t)MAX_THREADS;
    p.wgs = (unsigned)wgs; p.tiles = (int)std::min<int64_t>(own, INT32_MAX); p.join = (unsigned)(p.deep ? join * 8 : join);
    // Results, in waves of 32 rows: of up to `room` pieces where the row tiles are no more; else one of every row, and as many more as a cut into `room`
    // parts makes (rounded up, each row tile is one more than its share of them). Without shared positions only those of row tiles that are cut, each
    // of at least two pieces, which makes less than 2 room. There is room for them also where the row tiles stay whole, so that a workspace serves every
    // bound of the lengths and every window, and more of it never does with less.
    const int64_t piece_waves = a.shared ? ATT_BM / 32 : std::min<int64_t>(ATT_BM, most + 31) / 32;
    int64_t waves = piece_waves * room;
    if (tiles > room) {
        waves = piece_waves * room + own_waves + sh_tiles * (ATT_BM / 32);
        if (!a.shared) waves = std::min(waves, piece_waves * 2 * room);
    }
    p.most_waves = (int)waves;   // (with heads 2^27 at most: a call has no more than 2^30 rows)
    p.results = (size_t)waves * kv.heads;
    p.bytes = p.results * 32 * (kv.head_dim * 4 + 8) + (size_t)(own + 1) * sizeof(TreeTile) + 256;
    return p;
}

static int check_launch(const mmoe_attn_args &a, const TreePlan &p) {
    if (!p.fits) REFUSE("mmoe_attn_tree: %d sequences of up to %d positions, %d tokens, %d heads: too many for a launch", a.nseq, a.max_len, a.ntok, a.heads);
    return 0;
}

template <int T, int D, bool CAP, bool BIAS>
static int tree_run(const mmoe_attn_args &a, const mmoe_kv_cache &kv, const TreePlan &p, const uint64_t *bits, int words, int path) {
    TreeArgs A{};
    A.a = a; A.kv = kv;
    A.sh = log2_block(kv.block_size); A.group = a.heads / kv.heads;
    A.by_kv = divisor(kv.heads); A.by_group = divisor(A.group);
    A.s1 = CAP ? 2.0f * a.scale / a.cap * ATT_LOG2E : a.scale * ATT_LOG2E;
    A.s2 = a.cap * ATT_LOG2E;
    A.bits = bits; A.words = words; A.path = path;
    A.room = p.room; A.most_tiles = p.tiles; A.most_waves = p.most_waves;
    A.po = (float *)a.ws;
    A.pm = (float2 *)(A.po + p.results * 32 * D);
    A.tile_at = (TreeTile *)(A.pm + p.results * 32);
    if (p.many ? run(MMOE_K_ATT_TREE, k_attn_tree<T, D, CAP, BIAS, true>, p.wgs, 256, A) : run(MMOE_K_ATT_TREE, k_attn_tree<T, D, CAP, BIAS, false>, p.wgs, 256, A)) return -1;
    if (!p.room) return 0;
    return p.deep ? run(MMOE_K_ATT_TREE, k_tree_join<T, D, true>, p.join, 256, A) : run(MMOE_K_ATT_TREE, k_tree_join<T, D, false>, p.join, 256, A);
}
template <int T, int D>
static int tree_pick(const mmoe_attn_args &a, const mmoe_kv_cache &kv, const TreePlan &p, const uint64_t *b, int w, int path) {
    if (a.cap > 0) return a.slopes ? tree_run<T, D, true, true>(a, kv, p, b, w, path) : tree_run<T, D, true, false>(a, kv, p, b, w, path);
    return a.slopes ? tree_run<T, D, false, true>(a, kv, p, b, w, path) : tree_run<T, D, false, false>(a, kv, p, b, w, path);
}

// The layers' caches of a call that works on all of them
static int check_layers(const char *who, const mmoe_kv_cache *kv, int layers) {
    if (!kv) REFUSE("%s: no arguments", who);
    if (layers < 1 || layers > MMOE_KV_MAXLAYERS) REFUSE("%s: %d layers outside 1..%d", who, layers, MMOE_KV_MAXLAYERS);
    for (int i = 0; i < layers; i++) {
        const mmoe_kv_cache &c = kv[i];
        if (check_cache(who, &c)) return -1;
        if (c.head_dim < 8 || c.head_dim > 256 || c.head_dim % 8) REFUSE("%s: head_dim %d is not a multiple of 8 up to 256", who, c.head_dim);
        if (c.block_stride != kv->block_stride || c.head_stride != kv->head_stride || c.token_stride != kv->token_stride || c.nblocks != kv->nblocks ||
            c.block_size != kv->block_size || c.heads != kv->heads || c.head_dim != kv->head_dim || c.dtype != kv->dtype)
            REFUSE("%s: layer %d's cache is not like the first", who, i);
    }
    return 0;
}
static PageArgs page_args(const mmoe_kv_cache *kv, int layers) {
    PageArgs P{};
    P.kv = kv[0];
    P.sh = log2_block(kv->block_size);
    P.esize = kv->dtype == MMOE_F32 ? 4 : 2;
    P.pieces = kv->head_dim * P.esize / 16;
    P.all = P.pieces * kv->heads;
    P.by_pieces = divisor(P.pieces);
    for (int i = 0; i < layers; i++) { P.base[2 * i] = kv[i].k; P.base[2 * i + 1] = kv[i].v; }
    return P;
}

static int check_tables(const char *who, int nseq, int width, int nblocks, int block_size, int shared) {
    if (log2_block(block_size) < 0) REFUSE("%s: block size %d is not a power of two from 16 to 1024", who, block_size);
    if (nseq < 0 || nseq > MMOE_KV_MAXSEQ) REFUSE("%s: %d sequences outside 0..%d", who, nseq, MMOE_KV_MAXSEQ);
    if (nblocks < 0 || (int64_t)nblocks * block_size > INT32_MAX) REFUSE("%s: %d blocks of %d positions", who, nblocks, block_size);
    if (width < 1 || (int64_t)width * block_size > MAX_LEN) REFUSE("%s: tables of %d blocks of %d positions", who, width, block_size);
    if (shared < 0 || shared % block_size || shared / block_size > width) REFUSE("%s: %d shared positions (block size %d, %d blocks per table)", who, shared, block_size, width);
    return 0;
}

extern "C" {

int mmoe_tree_plan(const mmoe_tree_plan_args *p) {
    if (!p) REFUSE("mmoe_tree_plan: no arguments");
    const mmoe_tree_plan_args &a = *p;
    if (a.nseq < 0 || a.nseq > MMOE_KV_MAXSEQ) REFUSE("mmoe_tree_plan: %d sequences outside 0..%d", a.nseq, MMOE_KV_MAXSEQ);
    if (a.ntok < 0 || a.ntok > MAX_TOKENS) REFUSE("mmoe_tree_plan: %d tokens", a.ntok);
    if (a.words < 1 || a.words > MMOE_TREE_MAX / 64) REFUSE("mmoe_tree_plan: %d words of bits outside 1..%d", a.words, MMOE_TREE_MAX / 64);
    if (!a.ntok) return 0;
    if (!a.qstart || (a.nseq && !a.len) || !a.parent || !a.pos || !a.bits) REFUSE("mmoe_tree_plan: a pointer is missing");
    if (apart(a.bits, 8)) REFUSE("mmoe_tree_plan: bits must be aligned to 8 bytes");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    const int w = a.words, g = std::max(a.nseq, 1);   // (without sequences: one for the tokens of none)
    return w == 1 ? run(MMOE_K_TREE, k_tree_plan<1>, g, 64, a) : w == 2 ? run(MMOE_K_TREE, k_tree_plan<2>, g, 128, a)
         : w <= 4 ? run(MMOE_K_TREE, k_tree_plan<4>, g, 256, a) : run(MMOE_K_TREE, k_tree_plan<8>, g, 512, a);
}

size_t mmoe_attn_tree_ws(const mmoe_attn_args *p, const mmoe_kv_cache *kv, const uint64_t *bits, int words) {
    (void)bits;   // (what it points to does not count, nor whether it does)
    if (check_bits("mmoe_attn_tree", p, kv, words & ~MMOE_TREE_WINDOW)) return 0;
    const TreePlan pl = tree_plan(*p, *kv);
    return check_launch(*p, pl) ? 0 : pl.bytes;
}

int mmoe_attn_tree(const mmoe_attn_args *p, const mmoe_kv_cache *kv, const uint64_t *bits, int words) {
    const bool along = words & MMOE_TREE_WINDOW;
    words &= ~MMOE_TREE_WINDOW;
    if (check_bits("mmoe_attn_tree", p, kv, words)) return -1;
    const mmoe_attn_args &a = *p;
    if (!a.nseq || !a.ntok) return 0;
    if (!a.q || !a.out || !a.qstart || !a.len || !a.table || !bits) REFUSE("mmoe_attn_tree: a pointer is missing");
    if (apart(a.q, 16) || apart(a.out, 16)) REFUSE("mmoe_attn_tree: q and out must be aligned to 16 bytes");
    if (apart(bits, 8)) REFUSE("mmoe_attn_tree: bits must be aligned to 8 bytes");
    const TreePlan pl = tree_plan(a, *kv);
    if (check_launch(a, pl)) return -1;
    if (!a.ws || a.ws_bytes < pl.bytes || apart(a.ws, 256)) REFUSE("mmoe_attn_tree: workspace of %zu bytes (%zu needed, aligned to 256)", a.ws ? a.ws_bytes : 0, pl.bytes);
    if (mm_ready()) return -1;
    if (!a.max_q) return 0;   // no token is served
    OnDevice dev;
    if (!dev.ok) return -1;
    const int path = along && a.window ? a.window : INT32_MAX;
    if (kv->dtype == MMOE_F16) return kv->head_dim == 64 ? tree_pick<MMOE_F16, 64>(a, *kv, pl, bits, words, path) : tree_pick<MMOE_F16, 128>(a, *kv, pl, bits, words, path);
    return kv->head_dim == 64 ? tree_pick<MMOE_BF16, 64>(a, *kv, pl, bits, words, path) : tree_pick<MMOE_BF16, 128>(a, *kv, pl, bits, words, path);
}

int mmoe_tree_accept(const mmoe_tree_accept_args *p) {
    if (!p) REFUSE("mmoe_tree_accept: no arguments");
    const mmoe_tree_accept_args &a = *p;
    if (a.nseq < 0 || a.nseq > MMOE_KV_MAXSEQ) REFUSE("mmoe_tree_accept: %d sequences outside 0..%d", a.nseq, MMOE_KV_MAXSEQ);
    if (a.ntok < 0 || a.ntok > MAX_TOKENS) REFUSE("mmoe_tree_accept: %d tokens", a.ntok);
    if (!a.nseq) return 0;
    if (!a.qstart || !a.len || !a.count || !a.ctx || !a.last || (a.ntok && (!a.parent || !a.token || !a.next || !a.kept))) REFUSE("mmoe_tree_accept: a pointer is missing");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    return run(MMOE_K_TREE, k_tree_accept, a.nseq, 128, a);
}

int mmoe_kv_compact(const mmoe_kv_compact_args *p, const mmoe_kv_cache *kv, int layers) {
    if (!p) REFUSE("mmoe_kv_compact: no arguments");
    if (check_layers("mmoe_kv_compact", kv, layers)) return -1;
    const mmoe_kv_compact_args &a = *p;
    if (check_tables("mmoe_kv_compact", a.nseq, a.width, kv->nblocks, kv->block_size, 0)) return -1;
    if (a.nkept < 0 || a.nkept > MAX_LEN) REFUSE("mmoe_kv_compact: %d kept positions", a.nkept);
    if (!a.nseq || !a.nkept) return 0;
    if (!a.table || !a.first || !a.count || !a.kept) REFUSE("mmoe_kv_compact: a pointer is missing");
    const PageArgs P = page_args(kv, layers);
    // Short lists (a step's accepted tokens, a few of those that there is room for): a wave goes through one (64 sequences that drafted 64 tokens: 15.3 us,
    // by workgroups of 256 17.4; were 60 of them kept, 31 and 20). Else workgroups of 256 with as many pieces of a position, at least 128 bytes, as
    // leave 768 of them (4 sequences of 5000, 24 layers, 0.4 kept: 167 us, of 1024 threads 171); where there are not so many, of 1024 threads, from 160 on
    // (one sequence of 20000: 171 us, of 256 threads 194, with pieces of 64 bytes 207). A list goes through one workgroup per array and pieces, so that few
    // layers leave most of the card idle: of 20000 positions 6 layers 66 us (of 256 threads 115; 38 would be a copy's), one 37 (97; 6.4)
    const int64_t arrays = 2 * layers, lists = a.nseq * arrays;
    auto units_of = [&](int lanes) { return (P.all + lanes - 1) / lanes; };
    auto pieces_for = [&](int wgs) {
        int lanes = std::min(64, P.all);
        while (lanes > 8 && lists * units_of(lanes) < wgs) lanes = (lanes + 1) / 2;
        return lanes;
    };
    int threads = 64, lanes = std::min(64, P.all);
    if (a.nkept / a.nseq > 64) {
        threads = 256; lanes = pieces_for(768);
        if (lists * units_of(lanes) < 768) { threads = 1024; lanes = pieces_for(160); }
    }
    const int units = units_of(lanes);
    const int64_t wgs = lists * units;
    if (wgs * threads > (int64_t)MAX_THREADS) REFUSE("mmoe_kv_compact: %d sequences, %d layers, %d heads: too many for a launch", a.nseq, layers, kv->heads);
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    auto go = [&](auto kernel) { return run(MMOE_K_KV_PAGES, kernel, (unsigned)wgs, threads, a, P, lanes, units, divisor(lanes), divisor(units), divisor((uint32_t)arrays), (int)arrays); };
    return threads == 64 ? go(k_kv_compact<64>) : threads == 256 ? go(k_kv_compact<256>) : go(k_kv_compact<1024>);
}

int mmoe_kv_copy(const mmoe_kv_copy_args *p, const mmoe_kv_cache *kv, int layers) {
    if (!p) REFUSE("mmoe_kv_copy: no arguments");
    if (check_layers("mmoe_kv_copy", kv, layers)) return -1;
    const mmoe_kv_copy_args &a = *p;
    if (a.ncopy < 0 || a.ncopy > MMOE_KV_MAXSEQ) REFUSE("mmoe_kv_copy: %d copies outside 0..%d", a.ncopy, MMOE_KV_MAXSEQ);
    if (!a.ncopy) return 0;
    if (!a.copy_from || !a.copy_to) REFUSE("mmoe_kv_copy: a pointer is missing");
    const PageArgs P = page_args(kv, layers);
    const int64_t items = (int64_t)P.all * kv->block_size, units = (items + KY_T * KY_U - 1) / (KY_T * KY_U), wgs = units * a.ncopy * 2 * layers;
    if (wgs * KY_T > (int64_t)MAX_THREADS) REFUSE("mmoe_kv_copy: %d copies, %d layers, %d heads, blocks of %d: too many for a launch", a.ncopy, layers, kv->heads, kv->block_size);
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    return run(MMOE_K_KV_PAGES, k_kv_copy, (unsigned)wgs, KY_T, a, P, (int)units, divisor((uint32_t)units), divisor(2 * layers), 2 * layers);
}

int mmoe_kv_fork(const mmoe_kv_fork_args *p) {
    if (!p) REFUSE("mmoe_kv_fork: no arguments");
    const mmoe_kv_fork_args &a = *p;
    if (check_tables("mmoe_kv_fork", a.nseq, a.width, a.nblocks, a.block_size, a.shared)) return -1;
    if (a.nfork < 0 || a.nfork > MMOE_KV_MAXSEQ) REFUSE("mmoe_kv_fork: %d forks outside 0..%d", a.nfork, MMOE_KV_MAXSEQ);
    if (!a.nfree || !a.nfree_out || (a.nfork && (!a.src || !a.dst || !a.copy_from || !a.copy_to || !a.copy_count)) ||
        (a.nfork && a.nseq && (!a.ctx || !a.ctx_out || !a.table || !a.table_out)) || (a.nfork && a.nblocks && (!a.holders || !a.free_list)))
        REFUSE("mmoe_kv_fork: a pointer is missing");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    const int sh = log2_block(a.block_size);
    const bool one = (int64_t)a.nfork * a.width <= KO_ONE;
    if (a.nfork <= 1024 ? run(MMOE_K_KV_PAGES, k_kv_fork<1>, 1, 1024, a, sh, one, divisor(a.width)) : run(MMOE_K_KV_PAGES, k_kv_fork<4>, 1, 1024, a, sh, one, divisor(a.width))) return -1;
    return one || !a.nseq ? 0 : run(MMOE_K_KV_PAGES, k_kv_fork_rows, a.nfork, 256, a, sh);
}

int mmoe_kv_free(const mmoe_kv_free_args *p) {
    if (!p) REFUSE("mmoe_kv_free: no arguments");
    const mmoe_kv_free_args &a = *p;
    if (check_tables("mmoe_kv_free", a.nseq, a.width, a.nblocks, a.block_size, a.shared)) return -1;
    if ((int64_t)a.nseq * a.width > MAX_LEN) REFUSE("mmoe_kv_free: %d tables of %d blocks: more than 2^30 places", a.nseq, a.width);
    if (!a.nfree || !a.nfree_out || (a.nseq && (!a.ctx || !a.keep || !a.table || !a.len)) || (a.nblocks && !a.free_list)) REFUSE("mmoe_kv_free: a pointer is missing");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    const int sh = log2_block(a.block_size);
    return a.nseq <= 1024 ? run(MMOE_K_KV_PAGES, k_kv_free<1>, 1, a.nseq <= 256 ? 256 : 1024, a, sh) : run(MMOE_K_KV_PAGES, k_kv_free<4>, 1, 1024, a, sh);
}

}  // extern "C"
