// paged.hip -- the operators that serve many sequences at once (include/maplemoe.h, Part 3): argument checks and launches.
#include "paged_host.h"

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
    if (check_attn("mmoe_attn_paged", p, kv)) return 0;
    return att_plan(*p, *kv).bytes;
}

int mmoe_attn_paged(const mmoe_attn_args *p, const mmoe_kv_cache *kv) {
    if (check_attn("mmoe_attn_paged", p, kv)) return -1;
    return att_call<false>("mmoe_attn_paged", *p, kv);
}

}  // extern "C"
