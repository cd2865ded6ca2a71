// paged.hip -- the operators that serve many sequences at once (include/maplemoe.h, Part 3): argument checks and launches.
#include <hip/hip_runtime.h>
#include <math.h>
#include <algorithm>
#include <tuple>
#include <type_traits>
#include "ctx.h"
extern "C" {
#include "../../include/maplemoe.h"
}
#include "paged.h"

// One kernel on the library stream: the arguments converted to the kernel's parameter types and passed by address
template <typename... P, typename... A>
static int run(int kid, void (*f)(P...), dim3 g, dim3 b, A &&...a) {
    static_assert(sizeof...(P) == sizeof...(A), "kernel argument count");
    std::tuple<P...> v(static_cast<P>(a)...);
    void *ptr[sizeof...(P)];
    std::apply([&](auto &...x) { int i = 0; ((ptr[i++] = (void *)&x), ...); }, v);
    return mm_launch(kid, (const void *)f, g, b, ptr);
}

// The library's device current for the duration of a call
struct OnDevice {
    int prev = -1;
    bool ok = true;
    OnDevice() {
        int d = 0;
        ok = hipGetDevice(&d) == hipSuccess;
        if (ok && d != mm_device()) { prev = d; ok = hipSetDevice(mm_device()) == hipSuccess; }
        if (!ok) mm_error("device %d of the library cannot be made current", mm_device());
    }
    ~OnDevice() { if (prev >= 0) (void)hipSetDevice(prev); }
};

#define REFUSE(...) do { mm_error(__VA_ARGS__); return -1; } while (0)
#define MAX_LEN (1 << 30)      // positions of a sequence: positions and a tile's end are 32-bit integers everywhere
#define MAX_TOKENS (1 << 23)   // tokens of a call, of 256 threads each in a launch; with heads, 2^30 rows: a tile's end is a 32-bit integer too
#define MAX_CAP 1024           // its error is 2^-22 of it: below half a step of fp16 in the weights
#define MAX_THREADS 0xffffffffull   // of a launch
static bool apart(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; }
static int log2_block(int bs) {   // -1: not a block size
    for (int s = 4; s <= 10; s++) if (bs == 1 << s) return s;
    return -1;
}

static int check_cache(const char *who, const mmoe_kv_cache *c) {
    if (!c->k || !c->v || apart(c->k, 16) || apart(c->v, 16)) REFUSE("%s: cache pointers must be set and aligned to 16 bytes", who);
    if (c->dtype != MMOE_F32 && c->dtype != MMOE_F16 && c->dtype != MMOE_BF16) REFUSE("%s: cache type %d", who, c->dtype);
    if (log2_block(c->block_size) < 0) REFUSE("%s: block size %d is not a power of two from 16 to 1024", who, c->block_size);
    if (c->nblocks < 1 || (int64_t)c->nblocks * c->block_size > INT32_MAX) REFUSE("%s: %d blocks of %d positions", who, c->nblocks, c->block_size);
    if (c->heads < 1 || c->heads > 1024) REFUSE("%s: %d key/value heads", who, c->heads);
    if (c->block_stride < 0 || c->head_stride < 0 || c->token_stride < 0 || ((c->block_stride | c->head_stride | c->token_stride) & 7))
        REFUSE("%s: cache strides must be multiples of 8", who);
    if (c->token_stride < c->head_dim || c->token_stride > 1 << 26) REFUSE("%s: token stride %lld outside %d..%d", who, (long long)c->token_stride, c->head_dim, 1 << 26);
    return 0;
}

extern "C" {

int mmoe_kv_plan(const mmoe_kv_plan_args *p) {
    if (!p) REFUSE("mmoe_kv_plan: no arguments");
    const mmoe_kv_plan_args &a = *p;
    int sh = log2_block(a.block_size);
    if (sh < 0) REFUSE("mmoe_kv_plan: block size %d is not a power of two from 16 to 1024", a.block_size);
    if (a.nseq < 0 || a.nseq > MMOE_KV_MAXSEQ) REFUSE("mmoe_kv_plan: %d sequences outside 0..%d", a.nseq, MMOE_KV_MAXSEQ);
    if (a.ntok < 0 || a.ntok > MAX_TOKENS) REFUSE("mmoe_kv_plan: %d tokens", a.ntok);
    if (a.nblocks < 0 || (int64_t)a.nblocks * a.block_size > INT32_MAX) REFUSE("mmoe_kv_plan: %d blocks of %d positions", a.nblocks, a.block_size);
    if (a.width < 1 || (int64_t)a.width * a.block_size > MAX_LEN) REFUSE("mmoe_kv_plan: tables of %d blocks of %d positions", a.width, a.block_size);
    if (a.shared < 0 || a.shared % a.block_size || a.shared / a.block_size > a.width)
        REFUSE("mmoe_kv_plan: %d shared positions (block size %d, %d blocks per table)", a.shared, a.block_size, a.width);
    if (!a.nfree || !a.nfree_out || !a.qstart || (a.nseq && (!a.ctx || !a.add || !a.table || !a.len)) || (a.nblocks && !a.free_list) ||
        (a.ntok && (!a.pos || !a.slot)))
        REFUSE("mmoe_kv_plan: a pointer is missing");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    // The tokens in the same launch, or in one of their own over the whole card: 1000 tokens 6.0 / 8.8 us, 4000 7.4 / 8.9, 8000 8.3 / 8.2
    const bool one = a.ntok <= 4096;
    // 256 threads have fewer waves to wait for: 64 sequences 5.6 us, with 1024 threads 6.8
    const unsigned threads = std::max(a.nseq, a.ntok) <= 256 ? 256 : 1024;
    if (a.nseq <= 1024 ? run(MMOE_K_KV_PLAN, k_kv_plan<1>, 1, threads, a, sh, one) : run(MMOE_K_KV_PLAN, k_kv_plan<4>, 1, threads, a, sh, one)) return -1;
    return one ? 0 : run(MMOE_K_KV_PLAN, k_kv_tokens, (a.ntok + 255) / 256, 256, a, sh);
}

int mmoe_rope_freqs(int rot, double base, double factor, int orig, double slow, double fast, double *freq) {
    if (rot < 0 || rot > 256 || (rot & 1)) REFUSE("mmoe_rope_freqs: %d rotated dims", rot);
    if (!freq) REFUSE("mmoe_rope_freqs: no output");
    if (!(base > 1.0) || !(base < 1e300)) REFUSE("mmoe_rope_freqs: base %g", base);
    if (!(factor >= 1.0) || !(factor < 1e300)) REFUSE("mmoe_rope_freqs: factor %g", factor);
    if (orig < 0 || (orig > 0 && !(fast > slow && slow >= 0.0 && fast < 1e300))) REFUSE("mmoe_rope_freqs: orig %d, slow %g, fast %g", orig, slow, fast);
    for (int i = 0; i < rot / 2; i++) {
        double f = pow(base, -2.0 * i / rot), g = 0.0;
        if (orig > 0) {
            g = (orig * f / (2.0 * M_PI) - slow) / (fast - slow);
            g = g < 0.0 ? 0.0 : g > 1.0 ? 1.0 : g;
        }
        freq[i] = f * g + f / factor * (1.0 - g);
    }
    return 0;
}

}  // extern "C"

// ------------------------------------------------------------------------------------------------------
// Rotary positions
// ------------------------------------------------------------------------------------------------------
template <int IN, int OUT>
static int rope_launch(const mmoe_rope_args &a, const mmoe_kv_cache &kv, int cached, int sh) {
    // As many tokens per workgroup as RP_U heads per lane cover, once there are 512 workgroups: two tokens of 24 heads instead of one
    // 24.5 instead of 28.4 us at 8191 tokens, 7.7 instead of 8.9 at 2000; 6.8 instead of 6.5 at 1000
    const int nh = a.heads + a.kv_heads * (1 + cached), at_once = RP_U * RP_T / (a.head_dim / 8);
    const int tb = std::max(1, std::min(std::min(at_once / nh, RP_TB), a.ntok / 512));
    dim3 g((a.ntok + tb - 1) / tb);
    const bool pow2 = (a.head_dim & (a.head_dim - 1)) == 0;
    if (pow2 && a.interleaved) return run(MMOE_K_ROPE, k_rope<IN, OUT, RP_INTER>, g, RP_T, a, kv, cached, sh, tb);
    if (pow2 && a.rot % 16 == 0) return run(MMOE_K_ROPE, k_rope<IN, OUT, RP_SPLIT>, g, RP_T, a, kv, cached, sh, tb);
    return run(MMOE_K_ROPE, k_rope<IN, OUT, RP_ODD>, g, RP_T, a, kv, cached, sh, tb);
}
template <int IN>
static int rope_out(const mmoe_rope_args &a, const mmoe_kv_cache &kv, int cached, int sh) {
    return a.out_dtype == MMOE_F32 ? rope_launch<IN, MMOE_F32>(a, kv, cached, sh) : a.out_dtype == MMOE_F16 ? rope_launch<IN, MMOE_F16>(a, kv, cached, sh)
                                   : rope_launch<IN, MMOE_BF16>(a, kv, cached, sh);
}

// ------------------------------------------------------------------------------------------------------
// Attention
// ------------------------------------------------------------------------------------------------------
static int check_attn(const mmoe_attn_args *p, const mmoe_kv_cache *kv) {
    if (!p || !kv) REFUSE("mmoe_attn_paged: no arguments");
    const mmoe_attn_args &a = *p;
    if (check_cache("mmoe_attn_paged", kv)) return -1;
    if (kv->dtype == MMOE_F32) REFUSE("mmoe_attn_paged: cache type %d (fp16 or bf16)", kv->dtype);
    if (kv->head_dim != 64 && kv->head_dim != 128) REFUSE("mmoe_attn_paged: head_dim %d is not 64 or 128", kv->head_dim);
    if (a.heads < 1 || a.heads > 65535 || a.heads % kv->heads) REFUSE("mmoe_attn_paged: %d query heads over %d key/value heads", a.heads, kv->heads);
    if (a.nseq < 0 || a.nseq > MMOE_KV_MAXSEQ) REFUSE("mmoe_attn_paged: %d sequences outside 0..%d", a.nseq, MMOE_KV_MAXSEQ);
    if (a.ntok < 0 || a.ntok > MAX_TOKENS || (int64_t)a.ntok * a.heads > 1 << 30) REFUSE("mmoe_attn_paged: %d tokens", a.ntok);
    if (a.width < 1 || (int64_t)a.width * kv->block_size > MAX_LEN) REFUSE("mmoe_attn_paged: tables of %d blocks", a.width);
    if (a.max_q < 0 || a.max_len < 0 || a.max_len > (int64_t)a.width * kv->block_size)
        REFUSE("mmoe_attn_paged: max_q %d, max_len %d (tables of %d blocks)", a.max_q, a.max_len, a.width);
    if (a.shared < 0 || a.shared % kv->block_size || a.shared > a.max_len) REFUSE("mmoe_attn_paged: %d shared positions (block size %d, max_len %d)", a.shared, kv->block_size, a.max_len);
    if (a.window < 0) REFUSE("mmoe_attn_paged: window %d", a.window);
    if (!(a.scale >= 1e-20f) || !(a.scale <= 1e20f) || !(a.cap >= 0) || a.cap > MAX_CAP || (a.cap > 0 && !isfinite(4.0f * a.scale / a.cap))) REFUSE("mmoe_attn_paged: scale %g, cap %g", a.scale, a.cap);
    if (a.q_token < 0 || a.q_head < 0 || a.out_token < 0 || a.out_head < 0 || ((a.q_token | a.q_head | a.out_token | a.out_head) & 7))
        REFUSE("mmoe_attn_paged: strides must be multiples of 8");
    return 0;
}

// How a call is divided: row tiles, and runs or chunks of positions where the tiles alone are too few workgroups. Only the values in the
// arguments count (a captured call keeps its grid), and few of them: tokens, heads, the bounds. The numbers of workgroups are for the 256 compute
// units of the one device that the kernels are built and were measured for; a partition with fewer runs the same division in more turns.
struct AttPlan {
    int few, chunk, chunks, tiles, split, few_sh, tiles_sh, split_sh, parts;
    int64_t at_tile, at_few, entries, wgs, join_wgs;
    int join_all, join_few, join_threads;
    size_t bytes;
};
static AttPlan att_plan(const mmoe_attn_args &a, const mmoe_kv_cache &kv) {
    AttPlan p = {};
    const int group = a.heads / kv.heads;
    const int64_t rows = (int64_t)a.ntok * group, tiles = (rows + ATT_BM - 1) / ATT_BM, most_rows = (int64_t)std::min(a.max_q, a.ntok) * group;
    const int own = a.window && !a.hi ? (int)std::min<int64_t>(a.max_len - a.shared, (int64_t)a.window + a.max_q) : a.max_len - a.shared;
    // Runs of a row tile's positions: about 256 workgroups, half as many again where their runs stay above 512 positions (a second
    // workgroup on a CU adds a quarter to its rate, its partial results cost their bytes twice), none below 192. 960 rows over 40000
    // positions, 256 / 384 / 512 workgroups: 121 / 114 / 128 us; 256 rows over 16384: 31 / 38 / 56; 1200 over 20000: 85 / 74 / 89.
    // Runs of 256 / 512 / 1024 of 1000 positions: 20.1 / 22.9 / 25.7 us; one of 382 or two: 20.7 / 24.5. Tiles enough for one run each stay
    // whole: 3500 rows of 12 heads over up to 1100 positions 22.6 us, in two runs 33.
    auto runs = [&](int64_t groups, int positions) {
        const int64_t wgs = groups * kv.heads, n = (256 + wgs - 1) / wgs, n2 = (384 + wgs - 1) / wgs, most = positions / 192;
        return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(n > 1 && positions / n2 >= 512 ? n2 : n, most), ATT_PARTS / 2));
    };
    // Rows of a key/value head that k_attn_few takes: 16 are one product's, 32 over shared positions read them twice (from cache). So few
    // that all its workgroups are on the card at once start sooner than row tiles do: 46 rows, 2 heads, 5088 positions (120 workgroups)
    // 14.4 us, as row tiles 18.4; 36, 8, 3136 (312) 16.9, 18.4; but 228, 4, 1312 (360) 20.3, 18.6.
    p.few_sh = rows <= 32 || (rows + 15) / 16 * kv.heads * (a.shared / 256 + 1) <= 320;
    if (most_rows <= 16 || a.nseq > 1) p.few = 16;
    // Chunks: 1024 positions, down to 256 while there are fewer than 384 workgroups (one sequence of 100000: 256 50.5 us, 512 50.3, 1024 47.6,
    // 2048 47.9; 64 of up to 3000: 52.2, 49.6, 47.9, 62.5; 7 over 2048 shared: 128 12.9, 256 12.0, 512 13.9), and never more than ATT_PARTS / 2
    const int64_t units = (a.shared && p.few_sh ? (rows + 15) / 16 * (a.shared / 128) : 0) + (p.few ? a.nseq * (int64_t)(own / 128 + 1) : 0);
    p.chunk = 1024;
    while (p.chunk > 256 && units * kv.heads * 128 / p.chunk < 384) p.chunk >>= 1;
    p.chunk = std::max(p.chunk, (std::max(own, a.shared) / (ATT_PARTS / 2 - 1) + 128) & ~127);
    if (a.shared) {
        p.tiles_sh = p.few_sh ? (int)((rows + 15) / 16) : (int)tiles;
        p.split_sh = p.few_sh ? (a.shared + p.chunk - 1) / p.chunk : runs(tiles, a.shared);
    }
    p.split = 1;
    if (most_rows > p.few) {
        p.tiles = (int)tiles + a.nseq;
        // (with a window a tile sees that and its own tokens)
        p.split = runs(tiles, a.window && !a.hi ? (int)std::min<int64_t>(own, (int64_t)a.window + ATT_BM / group) : own);
    }
    if (p.few) {
        const int span = own + (a.window ? 31 : a.shared & 31);   // chunks begin at a multiple of 32
        // One chunk, and no join, beside row tiles that go over as many positions in one run: five prompts of up to 1100 tokens 21.8 us, with
        // a join of nothing 23.6; 8 sequences of 1 to 300 tokens over 1500 positions 40.7 and 40.6
        if (p.tiles && p.split == 1 && !p.split_sh && span <= 2048) p.chunk = std::max(128, (span + 127) & ~127);
        p.chunks = std::max(1, (span + p.chunk - 1) / p.chunk);
    }
    p.parts = p.split_sh + std::max(p.split, p.chunks);
    const int64_t all = (int64_t)a.ntok * a.heads;
    p.at_tile = p.split_sh * all;
    p.at_few = p.at_tile + (p.tiles && (p.split > 1 || p.split_sh) ? p.split * all : 0);
    p.entries = p.at_few + (p.few && (p.chunks > 1 || p.split_sh) ? (int64_t)p.chunks * a.nseq * 16 * kv.heads : 0);
    p.bytes = 256 + (size_t)p.entries * (kv.head_dim * 4 + 8);
    p.wgs = (int64_t)kv.heads * ((int64_t)p.tiles_sh * p.split_sh + (int64_t)p.tiles * p.split + (int64_t)p.chunks * a.nseq);
    p.join_few = !p.split_sh && p.tiles && p.split == 1;   // only sequences of few rows have partial results
    // A workgroup per row from 17 parts on (10 parts that way 81 us instead of 74 for the call; 32 parts in one lane group's registers 19
    // instead of 12), of 1024 threads from 129 on (390 parts: 162.3 us for the call, with 256 threads 164.6; 21 parts: 46, 34)
    p.join_all = p.parts > ATT_PER;
    p.join_threads = p.join_all && p.parts > 128 ? 1024 : 256;
    const int64_t jr = p.join_few ? 16ll * kv.heads * a.nseq : all, per = p.join_threads / (kv.head_dim / 4);
    p.join_wgs = p.join_all ? jr : (jr + per - 1) / per;
    return p;
}

// d > 0
static Div divisor(uint32_t d) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) l++;
    return Div{d, (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1), std::min(l, 1u), l ? l - 1 : 0};
}

template <int T, int D, bool CAP, bool BIAS>
static int att_run(const mmoe_attn_args &a, const mmoe_kv_cache &kv, const AttPlan &p) {
    AttArgs A{};
    A.a = a; A.kv = kv;
    A.sh = log2_block(kv.block_size); A.group = a.heads / kv.heads;
    A.n_sh = (unsigned)p.tiles_sh * p.split_sh * kv.heads;
    A.n_tile = (unsigned)p.tiles * p.split * kv.heads;
    A.n_few = (unsigned)p.chunks * a.nseq * kv.heads;
    A.tiles_sh = p.tiles_sh; A.tiles = p.tiles;
    A.by_heads = divisor(a.heads); A.by_kv = divisor(kv.heads); A.by_group = divisor(A.group);
    A.by_split = divisor(std::max(p.split, 1)); A.by_split_sh = divisor(std::max(p.split_sh, 1)); A.by_chunks = divisor(std::max(p.chunks, 1));
    A.sh_few = p.few_sh; A.few = p.few;
    A.split_sh = p.split_sh; A.split = p.split; A.chunk = p.chunk; A.chunks = p.chunks;
    A.parts_sh = p.split_sh;
    A.s1 = CAP ? 2.0f * a.scale / a.cap * ATT_LOG2E : a.scale * ATT_LOG2E;
    A.s2 = a.cap * ATT_LOG2E;
    A.pm = (float2 *)a.ws;
    A.po = (float *)((uint8_t *)a.ws + (size_t)(p.entries + 1) / 2 * 16);
    A.at_tile = p.at_tile; A.at_few = p.at_few;
    const dim3 g(A.n_sh + A.n_tile + A.n_few);
    const bool has_tiles = A.n_tile || (A.n_sh && !A.sh_few);
    if (!has_tiles ? run(MMOE_K_ATT_PAGED, k_attn_few<T, D, CAP, BIAS>, g, 256, A)
                   : run(MMOE_K_ATT_PAGED, k_attn_tile<T, D, CAP, BIAS>, g, 256, A)) return -1;
    if (p.parts == 1) return 0;
    return run(MMOE_K_ATT_PAGED, k_attn_join<T, D>, (unsigned)p.join_wgs, p.join_threads, A, p.join_all, p.join_few);
}
template <int T, int D>
static int att_pick(const mmoe_attn_args &a, const mmoe_kv_cache &kv, const AttPlan &p) {
    if (a.cap > 0) return a.slopes ? att_run<T, D, true, true>(a, kv, p) : att_run<T, D, true, false>(a, kv, p);
    return a.slopes ? att_run<T, D, false, true>(a, kv, p) : att_run<T, D, false, false>(a, kv, p);
}

extern "C" {

int mmoe_rope_kv(const mmoe_rope_args *p, const mmoe_kv_cache *kv) {
    if (!p) REFUSE("mmoe_rope_kv: no arguments");
    const mmoe_rope_args &a = *p;
    if (a.in_dtype < MMOE_F32 || a.in_dtype > MMOE_BF16 || a.out_dtype < MMOE_F32 || a.out_dtype > MMOE_BF16) REFUSE("mmoe_rope_kv: types %d, %d", a.in_dtype, a.out_dtype);
    if (a.head_dim < 8 || a.head_dim > 256 || a.head_dim % 8) REFUSE("mmoe_rope_kv: head_dim %d is not a multiple of 8 up to 256", a.head_dim);
    if (a.rot < 0 || a.rot > a.head_dim || (a.rot & 1)) REFUSE("mmoe_rope_kv: %d rotated dims of %d", a.rot, a.head_dim);
    if (a.ntok < 0 || a.ntok > MAX_TOKENS || a.heads < 0 || a.heads > 65535 || a.kv_heads < 0 || a.kv_heads > 1024) REFUSE("mmoe_rope_kv: %d tokens, %d heads, %d key/value heads", a.ntok, a.heads, a.kv_heads);
    if (!isfinite(a.mag)) REFUSE("mmoe_rope_kv: mag %g", a.mag);
    int sh = 0;
    if (kv) {
        if (check_cache("mmoe_rope_kv", kv)) return -1;
        if (kv->dtype != a.out_dtype || kv->heads != a.kv_heads || kv->head_dim != a.head_dim)
            REFUSE("mmoe_rope_kv: cache of %d heads of %d, type %d, for %d heads of %d, type %d", kv->heads, kv->head_dim, kv->dtype, a.kv_heads, a.head_dim, a.out_dtype);
        sh = log2_block(kv->block_size);
    }
    if (!a.ntok || (!a.heads && !a.kv_heads)) return 0;
    if (!a.pos || (a.rot && !a.freq) || (a.heads && (!a.q || !a.q_out)) || (a.kv_heads && !a.k) || (kv && (!a.v || !a.slot)) || (!kv && a.kv_heads && !a.k_out))
        REFUSE("mmoe_rope_kv: a pointer is missing");
    if (apart(a.q, 16) || apart(a.k, 16) || apart(a.v, 16) || apart(a.q_out, 16) || apart(a.k_out, 16)) REFUSE("mmoe_rope_kv: pointers must be aligned to 16 bytes");
    if ((a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head | a.qo_token | a.qo_head | a.ko_token | a.ko_head) & 7)
        REFUSE("mmoe_rope_kv: strides must be multiples of 8");
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    mmoe_kv_cache none = {};
    const mmoe_kv_cache &c = kv ? *kv : none;
    return a.in_dtype == MMOE_F32 ? rope_out<MMOE_F32>(a, c, kv != nullptr, sh) : a.in_dtype == MMOE_F16 ? rope_out<MMOE_F16>(a, c, kv != nullptr, sh)
                                  : rope_out<MMOE_BF16>(a, c, kv != nullptr, sh);
}

size_t mmoe_attn_paged_ws(const mmoe_attn_args *p, const mmoe_kv_cache *kv) {
    if (check_attn(p, kv)) return 0;
    return att_plan(*p, *kv).bytes;
}

int mmoe_attn_paged(const mmoe_attn_args *p, const mmoe_kv_cache *kv) {
    if (check_attn(p, kv)) return -1;
    const mmoe_attn_args &a = *p;
    if (!a.nseq || !a.ntok) return 0;
    if (!a.q || !a.out || !a.qstart || !a.len || !a.table) REFUSE("mmoe_attn_paged: a pointer is missing");
    if (apart(a.q, 16) || apart(a.out, 16)) REFUSE("mmoe_attn_paged: q and out must be aligned to 16 bytes");
    AttPlan pl = att_plan(a, *kv);
    if (pl.wgs * 256 > (int64_t)MAX_THREADS || pl.join_wgs * pl.join_threads > (int64_t)MAX_THREADS)
        REFUSE("mmoe_attn_paged: %d sequences of up to %d positions, %d tokens, %d heads: too many for a launch", a.nseq, a.max_len, a.ntok, a.heads);
    if (!a.ws || a.ws_bytes < pl.bytes || apart(a.ws, 256)) REFUSE("mmoe_attn_paged: workspace of %zu bytes (%zu needed, aligned to 256)", a.ws ? a.ws_bytes : 0, pl.bytes);
    if (mm_ready()) return -1;
    OnDevice dev;
    if (!dev.ok) return -1;
    if (kv->dtype == MMOE_F16) return kv->head_dim == 64 ? att_pick<MMOE_F16, 64>(a, *kv, pl) : att_pick<MMOE_F16, 128>(a, *kv, pl);
    return kv->head_dim == 64 ? att_pick<MMOE_BF16, 64>(a, *kv, pl) : att_pick<MMOE_BF16, 128>(a, *kv, pl);
}

}  // extern "C"
