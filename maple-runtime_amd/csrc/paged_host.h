// paged_host.h -- what the translation units of the operators for many sequences (paged.hip, drafts.hip) share on the host: argument checks,
// launches.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <algorithm>
#include <tuple>
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

// ------------------------------------------------------------------------------------------------------
// Attention
// ------------------------------------------------------------------------------------------------------
static int check_attn(const char *who, const mmoe_attn_args *p, const mmoe_kv_cache *kv) {
    if (!p || !kv) REFUSE("%s: no arguments", who);
    const mmoe_attn_args &a = *p;
    if (check_cache(who, kv)) return -1;
    if (kv->dtype == MMOE_F32) REFUSE("%s: cache type %d (fp16 or bf16)", who, kv->dtype);
    if (kv->head_dim != 64 && kv->head_dim != 128) REFUSE("%s: head_dim %d is not 64 or 128", who, kv->head_dim);
    if (a.heads < 1 || a.heads > 65535 || a.heads % kv->heads) REFUSE("%s: %d query heads over %d key/value heads", who, a.heads, kv->heads);
    if (a.nseq < 0 || a.nseq > MMOE_KV_MAXSEQ) REFUSE("%s: %d sequences outside 0..%d", who, a.nseq, MMOE_KV_MAXSEQ);
    if (a.ntok < 0 || a.ntok > MAX_TOKENS || (int64_t)a.ntok * a.heads > 1 << 30) REFUSE("%s: %d tokens", who, a.ntok);
    if (a.width < 1 || (int64_t)a.width * kv->block_size > MAX_LEN) REFUSE("%s: tables of %d blocks", who, a.width);
    if (a.max_q < 0 || a.max_len < 0 || a.max_len > (int64_t)a.width * kv->block_size)
        REFUSE("%s: max_q %d, max_len %d (tables of %d blocks)", who, a.max_q, a.max_len, a.width);
    if (a.shared < 0 || a.shared % kv->block_size || a.shared > a.max_len) REFUSE("%s: %d shared positions (block size %d, max_len %d)", who, a.shared, kv->block_size, a.max_len);
    if (a.window < 0) REFUSE("%s: window %d", who, a.window);
    if (!(a.scale >= 1e-20f) || !(a.scale <= 1e20f) || !(a.cap >= 0) || a.cap > MAX_CAP || (a.cap > 0 && !isfinite(4.0f * a.scale / a.cap))) REFUSE("%s: scale %g, cap %g", who, a.scale, a.cap);
    if (a.q_token < 0 || a.q_head < 0 || a.out_token < 0 || a.out_head < 0 || ((a.q_token | a.q_head | a.out_token | a.out_head) & 7))
        REFUSE("%s: strides must be multiples of 8", who);
    return 0;
}

// d > 0
static Div divisor(uint32_t d) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) l++;
    return Div{d, (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1), std::min(l, 1u), l ? l - 1 : 0};
}
