// paged.h -- kernels of the operators that serve many sequences at once (paged.hip): block tables and slot maps, rotary
// positions with the cache write, attention over the blocks.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) u4 gu4;   // 16 bytes of global memory (global_load, not flat_load)

// ------------------------------------------------------------------------------------------------------
// Types
// ------------------------------------------------------------------------------------------------------
template <int T> struct Elem;   // MMOE_F32, MMOE_F16, MMOE_BF16
template <> struct Elem<MMOE_F32> { static constexpr int size = 4; };
template <> struct Elem<MMOE_F16> { static constexpr int size = 2; };
template <> struct Elem<MMOE_BF16> { static constexpr int size = 2; };

template <int T> __device__ __forceinline__ float half_to_f(uint32_t bits) {   // the low 16 bits
    if (T == MMOE_BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half((unsigned short)bits));
}
// two values to a word of 16-bit ones, each rounded to nearest even
template <int T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (T == MMOE_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        b2 r = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, r);
    }
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
}
template <int T> __device__ __forceinline__ void load8(float *x, const void *p, int64_t at) {
    if (T == MMOE_F32) {
        const gu4 *q = (const gu4 *)((const float *)p + at);
        u4 a = q[0], b = q[1];
#pragma unroll
        for (int i = 0; i < 4; i++) { x[i] = __uint_as_float(a[i]); x[4 + i] = __uint_as_float(b[i]); }
    } else {
        u4 a = *(const gu4 *)((const uint16_t *)p + at);
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = half_to_f<T>(a[i] & 0xffff); x[2 * i + 1] = half_to_f<T>(a[i] >> 16); }
    }
}
template <int T> __device__ __forceinline__ void store8(void *p, int64_t at, const float *x) {
    if (T == MMOE_F32) {
        gu4 *q = (gu4 *)((float *)p + at);
        u4 a, b;
#pragma unroll
        for (int i = 0; i < 4; i++) { a[i] = __float_as_uint(x[i]); b[i] = __float_as_uint(x[4 + i]); }
        q[0] = a; q[1] = b;
    } else {
        u4 a;
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
        *(gu4 *)((uint16_t *)p + at) = a;
    }
}

// entries of the ascending a[0 .. n) that are <= v
__device__ __forceinline__ int count_le(const int *a, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        int m = (lo + hi) >> 1;
        if (a[m] <= v) lo = m + 1; else hi = m;
    }
    return lo;
}

// ------------------------------------------------------------------------------------------------------
// Block tables and slot maps (mmoe_kv_plan)
// ------------------------------------------------------------------------------------------------------
// Everything is a prefix sum over the sequences followed by flat loops (blocks given back, blocks taken, tokens) in which an
// item finds its sequence by a binary search of the sums in LDS, so one long sequence costs no more than many short ones.
// One workgroup holds it all: sums of up to 4096 sequences are 4 per thread, and the steps depend on each other through
// the free list. Bound: the latency of its dependent loads and barriers, not bytes (a step of 64 sequences moves 5 KB).
#define KP_T 1024

// exclusive prefix sums of a and b over the workgroup; totals in *ta, *tb. 64 bits: lengths come unchecked from the device.
__device__ __forceinline__ void scan2(long long &a, long long &b, long long *ta, long long *tb, long long (*red)[2]) {
    int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    long long x = a, y = b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        long long u = __shfl_up(x, d, 64), v = __shfl_up(y, d, 64);
        if (l >= d) { x += u; y += v; }
    }
    __syncthreads();   // red may still be read from the scan before
    if (l == 63) { red[w][0] = x; red[w][1] = y; }
    __syncthreads();
    long long p = 0, q = 0, tp = 0, tq = 0;
#pragma unroll
    for (int i = 0; i < KP_T / 64; i++) {
        if (i < w) { p += red[i][0]; q += red[i][1]; }
        tp += red[i][0]; tq += red[i][1];
    }
    a = p + x - a; b = q + y - b;
    *ta = tp; *tb = tq;
}

// position and slot of token t, whose sequence s the caller found; the tokens behind the last sequence get 0 and -1
__device__ __forceinline__ void kv_token(const mmoe_kv_plan_args &a, int sh, int t, int total, int s, int begin, int end) {
    int pos = 0, slot = -1;
    if (t < total) {
        pos = a.len[s] - (end - t);
        int blk = a.table[(int64_t)s * a.width + (pos >> sh)];
        if ((unsigned)blk < (unsigned)a.nblocks) slot = (blk << sh) + (pos & (a.block_size - 1));
    }
    a.pos[t] = pos; a.slot[t] = slot;
}

__global__ void __launch_bounds__(KP_T) k_kv_plan(mmoe_kv_plan_args a, int sh, int tokens) {
    __shared__ int start[MMOE_KV_MAXSEQ + 1], first[MMOE_KV_MAXSEQ + 1];
    __shared__ long long red[KP_T / 64][2];
    __shared__ int took[2];   // tokens and blocks of the sequences that fit
    const int tid = threadIdx.x, n = a.nseq, bs1 = a.block_size - 1, keep = a.shared >> sh;
    const int per = (n + KP_T - 1) / KP_T, s0 = tid * per;
    const long long room = (long long)a.width << sh;
    int ctx[MMOE_KV_MAXSEQ / KP_T], add[MMOE_KV_MAXSEQ / KP_T];
    bool fin[MMOE_KV_MAXSEQ / KP_T];
    if (tid < 2) took[tid] = 0;
    const int nfree0 = min(max(a.nfree[0], 0), a.nblocks);
#pragma unroll
    for (int i = 0; i < MMOE_KV_MAXSEQ / KP_T; i++) {
        bool in = i < per && s0 + i < n;
        ctx[i] = in ? a.ctx[s0 + i] : 0;
        add[i] = in ? a.add[s0 + i] : 0;
        fin[i] = in && a.done && a.done[s0 + i] != 0;
    }
    // 1. blocks given back, appended to the list
    int nfree = nfree0;
    if (a.done) {
        long long g = 0, z = 0, tg, tz;
#pragma unroll
        for (int i = 0; i < MMOE_KV_MAXSEQ / KP_T; i++)
            if (fin[i]) g += max((int)((min((long long)max(ctx[i], 0), room) + bs1) >> sh) - keep, 0);
        scan2(g, z, &tg, &tz, red);
#pragma unroll
        for (int i = 0; i < MMOE_KV_MAXSEQ / KP_T; i++) {
            if (i < per && s0 + i < n) first[s0 + i] = (int)min(g, (long long)a.nblocks);
            if (fin[i]) g += max((int)((min((long long)max(ctx[i], 0), room) + bs1) >> sh) - keep, 0);
        }
        __syncthreads();
        int back = (int)min(tg, (long long)(a.nblocks - nfree0));
        for (int j = tid; j < back; j += KP_T) {
            int s = count_le(first, n, j) - 1;
            a.free_list[nfree0 + j] = a.table[(int64_t)s * a.width + keep + j - first[s]];
        }
        nfree += back;
    }
    // 2. the sequences that fit: a prefix, since both sums only grow (one that cannot fit counts more tokens than there is room for)
    long long need[MMOE_KV_MAXSEQ / KP_T], tok[MMOE_KV_MAXSEQ / KP_T], cn = 0, ct = 0, tn, tt;
#pragma unroll
    for (int i = 0; i < MMOE_KV_MAXSEQ / KP_T; i++) {
        if (fin[i]) ctx[i] = min(ctx[i], a.shared);
        long long c = ctx[i], e = c + add[i];
        bool ok = c >= 0 && add[i] >= 0 && e <= room;
        need[i] = ok && add[i] > 0 ? ((e + bs1) >> sh) - ((c + bs1) >> sh) : 0;
        tok[i] = ok ? add[i] : (long long)a.ntok + 1;
        if (i >= per || s0 + i >= n) tok[i] = 0;
        cn += need[i]; ct += tok[i];
    }
    scan2(cn, ct, &tn, &tt, red);
    unsigned fits = 0;
#pragma unroll
    for (int i = 0; i < MMOE_KV_MAXSEQ / KP_T; i++) {
        if (i >= per || s0 + i >= n) continue;
        first[s0 + i] = (int)min(cn, (long long)a.nblocks + 1);
        start[s0 + i] = (int)min(ct, (long long)a.ntok);
        cn += need[i]; ct += tok[i];
        if (cn <= nfree && ct <= a.ntok) {
            fits |= 1u << i;
            atomicMax(&took[0], (int)ct); atomicMax(&took[1], (int)cn);
        }
    }
    __syncthreads();
    const int total = took[0], blocks = took[1];
#pragma unroll
    for (int i = 0; i < MMOE_KV_MAXSEQ / KP_T; i++) {
        if (i >= per || s0 + i >= n) continue;
        bool f = (fits >> i) & 1;
        if (!f) { start[s0 + i] = total; first[s0 + i] = blocks; add[i] = 0; }
        a.qstart[s0 + i] = start[s0 + i];
        a.len[s0 + i] = ctx[i] + add[i];
    }
    if (tid == 0) { start[n] = total; a.qstart[n] = total; a.nfree_out[0] = nfree - blocks; }
    __syncthreads();   // also: the list's appended entries and len are written
    // 3. new blocks, from the end of the list; then the tokens
    for (int j = tid; j < blocks; j += KP_T) {
        int s = count_le(first, n, j) - 1;
        int held = (a.len[s] - (start[s + 1] - start[s]) + bs1) >> sh;
        a.table[(int64_t)s * a.width + held + j - first[s]] = a.free_list[nfree - 1 - j];
    }
    if (!tokens) return;
    __syncthreads();
    for (int t = tid; t < a.ntok; t += KP_T) {
        int s = max(count_le(start, n, t) - 1, 0);
        kv_token(a, sh, t, total, s, start[s], start[s + 1]);
    }
}

// The tokens of a large step, in a launch of their own over the whole card
__global__ void __launch_bounds__(256) k_kv_tokens(mmoe_kv_plan_args a, int sh) {
    __shared__ int start[MMOE_KV_MAXSEQ + 1];
    for (int i = threadIdx.x; i <= a.nseq; i += 256) start[i] = a.qstart[i];
    __syncthreads();
    for (int t = blockIdx.x * 256 + threadIdx.x; t < a.ntok; t += gridDim.x * 256) {
        int s = max(count_le(start, a.nseq, t) - 1, 0);
        kv_token(a, sh, t, start[a.nseq], s, start[s], start[s + 1]);
    }
}

// ------------------------------------------------------------------------------------------------------
// Rotary positions and the cache write (mmoe_rope_kv)
// ------------------------------------------------------------------------------------------------------
// A workgroup takes tb tokens: their cos / sin into LDS once for all heads, then the heads in units of 8 values. The angle is
// reduced to half turns in 64 bits (pos * freq reaches 1e6 radians, where 32 bits are 0.06 off) before the 32-bit sine.
#define RP_T 256
#define RP_HALF 128   // largest rot / 2
#define RP_TB 8       // most tokens per workgroup
enum { RP_INTER, RP_SPLIT, RP_ODD };   // pairs (2 i, 2 i + 1); (i, i + rot / 2) with rot / 2 in whole units of 8, or not

__device__ __forceinline__ void rope_angles(const mmoe_rope_args &a, int t0, int nt, float2 *cs) {
    const int half = a.rot >> 1;
    for (int j = threadIdx.x; j < nt * half; j += RP_T) {
        int t = j / half, i = j - t * half;
        double h = (double)a.pos[t0 + t] * (a.freq[i] * 0.318309886183790671538);   // half turns
        h -= 2.0 * __builtin_rint(h * 0.5);
        float s, c;
        sincospif((float)h, &s, &c);
        cs[t * RP_HALF + i] = make_float2(c * a.mag, s * a.mag);
    }
}

// Head hd of a token's query heads | key heads | value heads (the last with a cache only): where it comes from and goes to.
struct RopeHead {
    const void *in; void *out;
    int64_t src, dst;
    bool turn, live;
};
__device__ __forceinline__ RopeHead rope_head(const mmoe_rope_args &a, const mmoe_kv_cache &kv, int cached, int sh, int64_t tok, int hd) {
    RopeHead r;
    r.live = true;
    int64_t slot = 0;
    if (cached) {
        int s = a.slot[tok];
        r.live = s >= 0 && (s >> sh) < kv.nblocks;
        slot = (int64_t)(s >> sh) * kv.block_stride + (int64_t)(s & (kv.block_size - 1)) * kv.token_stride;
    }
    int hk = hd - a.heads, hv = hk - a.kv_heads;
    r.turn = hv < 0;
    if (hk < 0) { r.in = a.q; r.src = tok * a.q_token + hd * a.q_head; r.out = a.q_out; r.dst = tok * a.qo_token + hd * a.qo_head; }
    else if (hv < 0) {
        r.in = a.k; r.src = tok * a.k_token + hk * a.k_head;
        r.out = cached ? kv.k : a.k_out;
        r.dst = cached ? slot + hk * kv.head_stride : tok * a.ko_token + hk * a.ko_head;
    } else { r.in = a.v; r.src = tok * a.v_token + hv * a.v_head; r.out = kv.v; r.dst = slot + hv * kv.head_stride; }
    return r;
}

template <int IN, int OUT, int LAY>
__global__ void __launch_bounds__(RP_T) k_rope(mmoe_rope_args a, mmoe_kv_cache kv, int cached, int sh, int tb) {
    __shared__ float2 cs[RP_TB * RP_HALF];
    __shared__ float row[LAY == RP_ODD ? RP_T * 8 : 1];
    const int t0 = blockIdx.x * tb, nt = min(tb, a.ntok - t0), half = a.rot >> 1, dc = a.head_dim >> 3;
    const int nh = a.heads + a.kv_heads + (cached ? a.kv_heads : 0), all = nt * nh;   // heads of the workgroup's tokens
    rope_angles(a, t0, nt, cs);
    __syncthreads();
    if (LAY == RP_ODD) {
        // the round's heads through LDS: a unit's partners start anywhere in another unit
        const int hpr = RP_T / dc, hl = threadIdx.x / dc, d0 = (threadIdx.x - hl * dc) * 8;
        for (int j0 = 0; j0 < all; j0 += hpr) {
            int j = j0 + hl, t = j / nh;
            bool on = hl < hpr && j < all;
            RopeHead r;
            float x[8], y[8], *mine = row + threadIdx.x * 8, *head = row + hl * a.head_dim;
            if (on) {
                r = rope_head(a, kv, cached, sh, t0 + t, j - t * nh);
                on = r.live;
            }
            if (on) {
                load8<IN>(x, r.in, r.src + d0);
#pragma unroll
                for (int i = 0; i < 8; i++) mine[i] = x[i];
            }
            __syncthreads();
            if (on) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    int d = d0 + i;
                    y[i] = x[i];
                    if (!r.turn || d >= a.rot) continue;
                    float2 c = cs[t * RP_HALF + (d < half ? d : d - half)];
                    y[i] = d < half ? fmaf(x[i], c.x, -(head[d + half] * c.y)) : fmaf(x[i], c.x, head[d - half] * c.y);
                }
                store8<OUT>(r.out, r.dst + d0, y);
            }
            __syncthreads();
        }
        return;
    }
    for (int j = threadIdx.x; j < all * dc; j += RP_T) {
        int hd = j / dc, d0 = (j - hd * dc) * 8, t = hd / nh;
        RopeHead r = rope_head(a, kv, cached, sh, t0 + t, hd - t * nh);
        if (!r.live) continue;
        const float2 *w = cs + t * RP_HALF;
        float x[8], y[8];
        if (!r.turn || d0 >= a.rot) {
            load8<IN>(x, r.in, r.src + d0);
            store8<OUT>(r.out, r.dst + d0, x);
        } else if (LAY == RP_INTER) {
            load8<IN>(x, r.in, r.src + d0);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                bool in = d0 + i < a.rot;
                float2 c = in ? w[(d0 + i) >> 1] : make_float2(1.0f, 0.0f);
                y[i] = in ? fmaf(x[i], c.x, -(x[i + 1] * c.y)) : x[i];
                y[i + 1] = in ? fmaf(x[i + 1], c.x, x[i] * c.y) : x[i + 1];
            }
            store8<OUT>(r.out, r.dst + d0, y);
        } else if (d0 < half) {   // the first half's unit takes its partner along: in place, none may read what another has written
            float z[8];
            load8<IN>(x, r.in, r.src + d0);
            load8<IN>(z, r.in, r.src + d0 + half);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float2 c = w[d0 + i];
                y[i] = fmaf(x[i], c.x, -(z[i] * c.y));
                z[i] = fmaf(z[i], c.x, x[i] * c.y);
            }
            store8<OUT>(r.out, r.dst + d0, y);
            store8<OUT>(r.out, r.dst + d0 + half, z);
        }
    }
}

// ------------------------------------------------------------------------------------------------------
// Attention over the blocks (mmoe_attn_paged)
// ------------------------------------------------------------------------------------------------------
struct AttArgs {
    mmoe_attn_args a;
    mmoe_kv_cache kv;
    int sh, group;   // log2 of the block size, query heads per key/value head
};

// A wave per (token, query head): 64 positions at a time, one per lane for the scores, dims over lanes for the values.
template <int T, int D>
__global__ void __launch_bounds__(64) k_attn_simple(AttArgs A) {
    const mmoe_attn_args &a = A.a;
    __shared__ float qs[D], ps[64];
    __shared__ int64_t ofs[64];
    int t = blockIdx.x, h = blockIdx.y, l = threadIdx.x;
    if (t >= a.qstart[a.nseq]) return;
    int s = max(count_le(a.qstart, a.nseq, t) - 1, 0), len = a.len[s], pos = len - (a.qstart[s + 1] - t);
    if (t - a.qstart[s] >= a.max_q) return;
    int lo = a.lo ? a.lo[t] : 0, hi = a.hi ? a.hi[t] : pos + 1;
    if (a.window > 0) lo = max(lo, pos - a.window);
    lo = max(lo, 0); hi = min(min(hi, len), a.max_len);
    for (int d = l; d < D; d += 64) qs[d] = half_to_f<T>(((const uint16_t *)a.q)[t * a.q_token + h * a.q_head + d]);
    __syncthreads();
    float m = -__builtin_inff(), sum = 0, o[D / 64] = {};
    for (int p0 = lo; p0 < hi; p0 += 64) {
        int p = p0 + l, blk = -1;
        if (p < hi) blk = a.table[(int64_t)s * a.width + (p >> A.sh)];
        bool see = (unsigned)blk < (unsigned)A.kv.nblocks;
        int64_t at = see ? blk * A.kv.block_stride + (h / A.group) * A.kv.head_stride + (p & (A.kv.block_size - 1)) * A.kv.token_stride : 0;
        float x = -__builtin_inff();
        if (see) {
            float v = 0;
            for (int d = 0; d < D; d += 8) {
                float k[8];
                load8<T>(k, A.kv.k, at + d);
                for (int i = 0; i < 8; i++) v = fmaf(k[i], qs[d + i], v);
            }
            x = v * a.scale;
            if (a.cap > 0) x = a.cap * tanhf(x / a.cap);
            if (a.slopes) x -= a.slopes[h] * (float)abs(pos - p);
        }
        float mx = x;
        for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        float mn = fmaxf(m, mx), base = mn == -__builtin_inff() ? 0 : mn, alpha = expf(m - base), e = see ? expf(x - base) : 0;
        m = mn;
        ps[l] = e; ofs[l] = see ? at : -1;
        float es = e;
        for (int d = 1; d < 64; d <<= 1) es += __shfl_xor(es, d, 64);
        sum = sum * alpha + es;
        __syncthreads();
        for (int i = 0; i < D / 64; i++) o[i] *= alpha;
        for (int j = 0; j < 64; j++) {
            if (ofs[j] < 0) continue;
            for (int i = 0; i < D / 64; i++) o[i] = fmaf(ps[j], half_to_f<T>(((const uint16_t *)A.kv.v)[ofs[j] + l + 64 * i]), o[i]);
        }
        __syncthreads();
    }
    for (int i = 0; i < D / 64; i++)
        ((uint16_t *)a.out)[t * a.out_token + h * a.out_head + l + 64 * i] = (uint16_t)pack2<T>(sum == 0 ? 0.0f : o[i] / sum, 0);
    if (a.lse && l == 0) a.lse[(int64_t)t * a.heads + h] = sum == 0 ? -__builtin_inff() : m + logf(sum);
}
