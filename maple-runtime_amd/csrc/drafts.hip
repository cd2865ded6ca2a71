// drafts.hip -- drafted tokens and shared blocks (include/maplemoe.h, Part 3): argument checks and launches.
#include "paged_host.h"
#include "drafts.h"

static int check_bits(const char *who, const mmoe_attn_args *p, const mmoe_kv_cache *kv, int words) {
    if (check_attn(who, p, kv)) return -1;
    if (p->hi) REFUSE("%s: hi is set (new tokens are seen by their bits)", who);
    if (words < 1 || words > MMOE_TREE_MAX / 64) REFUSE("%s: %d words of bits outside 1..%d", who, words, MMOE_TREE_MAX / 64);
    if (p->max_q > 64 * words) REFUSE("%s: max_q %d for %d words of bits", who, p->max_q, words);
    return 0;
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
    (void)bits;
    if (check_bits("mmoe_attn_tree", p, kv, words)) return 0;
    return att_plan(*p, *kv).bytes;
}

int mmoe_attn_tree(const mmoe_attn_args *p, const mmoe_kv_cache *kv, const uint64_t *bits, int words) {
    if (check_bits("mmoe_attn_tree", p, kv, words)) return -1;
    if (apart(bits, 8)) REFUSE("mmoe_attn_tree: bits must be aligned to 8 bytes");
    return att_call<true>("mmoe_attn_tree", *p, kv, bits, words);
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
    int lanes = std::min(64, P.all);
    while (lanes > 8 && (int64_t)a.nseq * 2 * layers * ((P.all + lanes - 1) / lanes) < 768) lanes = (lanes + 1) / 2;
    const int units = (P.all + lanes - 1) / lanes;
    const int64_t wgs = (int64_t)a.nseq * 2 * layers * units;
    if (wgs * KC_T > (int64_t)MAX_THREADS) REFUSE("mmoe_kv_compact: %d sequences, %d layers, %d heads: too many for a launch", a.nseq, layers, kv->heads);
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    return run(MMOE_K_KV_PAGES, k_kv_compact, (unsigned)wgs, KC_T, a, P, lanes, units, divisor(lanes), divisor(units), divisor(2 * layers), 2 * layers);
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
    const bool one = (int64_t)a.nfork * a.width <= 4096;
    if (a.nfork <= 1024 ? run(MMOE_K_KV_PAGES, k_kv_fork<1>, 1, 1024, a, sh, one) : run(MMOE_K_KV_PAGES, k_kv_fork<4>, 1, 1024, a, sh, one)) return -1;
    return one || !a.nseq ? 0 : run(MMOE_K_KV_PAGES, k_kv_fork_rows, a.nfork, 256, a, sh);
}

int mmoe_kv_free(const mmoe_kv_free_args *p) {
    if (!p) REFUSE("mmoe_kv_free: no arguments");
    const mmoe_kv_free_args &a = *p;
    if (check_tables("mmoe_kv_free", a.nseq, a.width, a.nblocks, a.block_size, a.shared)) return -1;
    if (!a.nfree || !a.nfree_out || (a.nseq && (!a.ctx || !a.keep || !a.table || !a.len)) || (a.nblocks && !a.free_list)) REFUSE("mmoe_kv_free: a pointer is missing");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    const int sh = log2_block(a.block_size);
    return a.nseq <= 1024 ? run(MMOE_K_KV_PAGES, k_kv_free<1>, 1, 1024, a, sh) : run(MMOE_K_KV_PAGES, k_kv_free<4>, 1, 1024, a, sh);
}

}  // extern "C"
