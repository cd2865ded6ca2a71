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
// eight values as they lie in memory
template <int T> struct Raw8 { u4 w[T == MMOE_F32 ? 2 : 1]; };
template <int T> __device__ __forceinline__ Raw8<T> load8(const void *p, int64_t at) {
    const gu4 *q = (const gu4 *)((const uint8_t *)p + at * Elem<T>::size);
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < Elem<T>::size / 2; i++) r.w[i] = q[i];
    return r;
}
template <int T> __device__ __forceinline__ void unpack8(float *x, const Raw8<T> &r) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (T == MMOE_F32) { x[i] = __uint_as_float(r.w[0][i]); x[4 + i] = __uint_as_float(r.w[Elem<T>::size / 4][i]); }
        else { x[2 * i] = half_to_f<T>(r.w[0][i] & 0xffff); x[2 * i + 1] = half_to_f<T>(r.w[0][i] >> 16); }
    }
}
template <int T> __device__ __forceinline__ void store8(void *p, const float *x) {
    if (T == MMOE_F32) {
        gu4 *q = (gu4 *)p;
        u4 a, b;
#pragma unroll
        for (int i = 0; i < 4; i++) { a[i] = __float_as_uint(x[i]); b[i] = __float_as_uint(x[4 + i]); }
        q[0] = a; q[1] = b;
    } else {
        u4 a;
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
        *(gu4 *)p = a;
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

// the number of i in 0 .. n - 1 for which f holds, by a wave for one f: every load under way at once instead of a search's one by one
template <typename F> __device__ __forceinline__ int count_wave(int n, F &&f) {
    int c = 0;
    for (int i = 0; i < n; i += 64) {
        int j = i + (threadIdx.x & 63);
        c += __popcll(__ballot(j < n && f(j)));
    }
    return c;
}

template <typename F> __device__ __forceinline__ int wave_reduce(int v, F &&f) {   // in registers: an exchange through LDS costs 100 cycles a step
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0xb1, 15, 15, false));    // lane ^ 1
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x4e, 15, 15, false));    // lane ^ 2
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 15, 15, false));   // mirrored in 8
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 15, 15, false));   // mirrored in 16
    auto a = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    v = f((int)a[0], (int)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return __builtin_amdgcn_readfirstlane(f((int)b[0], (int)b[1]));
}
__device__ __forceinline__ int wave_min(int v) { return wave_reduce(v, [](int x, int y) { return min(x, y); }); }
__device__ __forceinline__ int wave_max(int v) { return wave_reduce(v, [](int x, int y) { return max(x, y); }); }

// ------------------------------------------------------------------------------------------------------
// Block tables and slot maps (mmoe_kv_plan)
// ------------------------------------------------------------------------------------------------------
// Everything is a prefix sum over the sequences followed by flat loops (blocks given back, blocks taken, tokens) in which an
// item finds its sequence by a binary search of the sums in LDS, so one long sequence costs no more than many short ones. One
// workgroup holds it all, since the steps depend on each other through the free list. Bound: the latency of dependent loads
// (lengths; a table's begun block and the list's end; the stores), not bytes (a step of 64 sequences moves 5 KB), so what a later step
// needs is loaded as soon as its address is known and kept in LDS. Measured: 64 sequences of one token, 3 finished, 6.2 us (12.3 with
// what is taken and given back read from memory again, 9.4 with the totals by atomics in LDS); 301 prompts of up to 400 tokens 7.0 us.
#define KP_LIM (1 << 30)     // sums stop here: above every count there is room for, and two of them still fit
#define KP_TOP 1024          // list entries and the like kept in LDS

// inclusive sums over a wave, stopping at KP_LIM (a sum that has stopped stays, so the order of the additions does not matter)
__device__ __forceinline__ unsigned scan_wave(unsigned v) {
#define KP_STEP(ctrl, rows) v = min(v + (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 15, false), (unsigned)KP_LIM)
    KP_STEP(0x111, 15); KP_STEP(0x112, 15); KP_STEP(0x114, 15); KP_STEP(0x118, 15);   // from 1, 2, 4, 8 lanes below in the row of 16
    KP_STEP(0x142, 10); KP_STEP(0x143, 12);                                          // the row before's last, the first half's last
#undef KP_STEP
    return v;
}
// exclusive sums of a and b over the workgroup, and their totals
__device__ __forceinline__ void scan2(unsigned &a, unsigned &b, unsigned *ta, unsigned *tb, uint2 *red) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const unsigned x = scan_wave(a), y = scan_wave(b);
    __syncthreads();   // red may still be read from the scan before
    if (l == 63) red[w] = make_uint2(x, y);
    __syncthreads();
    unsigned p = 0, q = 0, tp = 0, tq = 0;
    for (int i = 0; i < nw; i++) {
        uint2 r = red[i];
        if (i < w) { p = min(p + r.x, (unsigned)KP_LIM); q = min(q + r.y, (unsigned)KP_LIM); }
        tp = min(tp + r.x, (unsigned)KP_LIM); tq = min(tq + r.y, (unsigned)KP_LIM);
    }
    // the lanes below this one (a difference would not undo a sum that has stopped)
    unsigned ex = (unsigned)__shfl_up((int)x, 1, 64), ey = (unsigned)__shfl_up((int)y, 1, 64);
    if (l == 0) ex = ey = 0;
    a = min(p + ex, (unsigned)KP_LIM); b = min(q + ey, (unsigned)KP_LIM);
    *ta = tp; *tb = tq;
}

// PER: consecutive sequences of a thread
template <int PER>
__global__ void __launch_bounds__(1024) k_kv_plan(mmoe_kv_plan_args a, int sh, int tokens) {
    constexpr int NS = PER * 1024;
    __shared__ int start[NS + 1], first[NS + 1], lens[NS], tail[NS], given[KP_TOP], top[KP_TOP];
    __shared__ uint2 red[16];
    const int tid = threadIdx.x, nt = blockDim.x, n = a.nseq, bs1 = a.block_size - 1, keep = a.shared >> sh, s0 = tid * PER;
    const int room = a.width << sh;   // < 2^31
    int ctx[PER], add[PER], old[PER];
    bool fin[PER];
    const int nfree0 = min(max(a.nfree[0], 0), a.nblocks);
    for (int j = tid; j < min(nfree0, KP_TOP); j += nt) top[j] = a.free_list[nfree0 - 1 - j];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const bool in = s0 + i < n;
        ctx[i] = in ? a.ctx[s0 + i] : 0;
        add[i] = in ? a.add[s0 + i] : 0;
        fin[i] = in && a.done && a.done[s0 + i] != 0;
    }
    // the block that a sequence has begun
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (fin[i]) old[i] = max((min(max(ctx[i], 0), room) + bs1 >> sh) - keep, 0);   // to be given back
        else old[i] = 0;
        if (fin[i]) ctx[i] = min(ctx[i], a.shared);
        const int at = ctx[i] >> sh;
        if (s0 + i < n) tail[s0 + i] = ctx[i] > 0 && (ctx[i] & bs1) && at < a.width ? a.table[(int64_t)(s0 + i) * a.width + at] : -1;
    }
    // 1. blocks given back, appended to the list
    int nfree = nfree0;
    if (a.done) {
        unsigned g = 0, z = 0, tg, tz;
#pragma unroll
        for (int i = 0; i < PER; i++) g = min(g + old[i], (unsigned)KP_LIM);
        scan2(g, z, &tg, &tz, red);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (s0 + i < n) first[s0 + i] = (int)min(g, (unsigned)a.nblocks);
            g = min(g + old[i], (unsigned)KP_LIM);
        }
        __syncthreads();
        const int back = (int)min(tg, (unsigned)(a.nblocks - nfree0));
        for (int j = tid; j < back; j += nt) {
            int s = count_le(first, n, j) - 1;
            const int b = a.table[(int64_t)s * a.width + keep + j - first[s]];
            a.free_list[nfree0 + j] = b;
            if (j < KP_TOP) given[j] = b;
        }
        nfree += back;   // (scan2 waits for given, and for what is only in memory)
    }
    auto taken = [&](int j) {   // the j-th block from the end of the list
        const int at = nfree - 1 - j, g = at - nfree0;
        return g >= 0 ? g < KP_TOP ? given[g] : a.free_list[at] : -g - 1 < KP_TOP ? top[-g - 1] : a.free_list[at];
    };
    // 2. the sequences that fit: a prefix, since both sums only grow (one that cannot fit counts more tokens than there is room for)
    unsigned need[PER], tok[PER], cn = 0, ct = 0, tn, tt;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const long long e = (long long)ctx[i] + add[i];
        const bool ok = ctx[i] >= 0 && add[i] >= 0 && e <= room;
        need[i] = ok && add[i] > 0 ? (unsigned)(((e + bs1) >> sh) - (((long long)ctx[i] + bs1) >> sh)) : 0;
        tok[i] = ok ? min((unsigned)add[i], (unsigned)KP_LIM) : (unsigned)KP_LIM;
        if (s0 + i >= n) tok[i] = 0;
        cn = min(cn + need[i], (unsigned)KP_LIM); ct = min(ct + tok[i], (unsigned)KP_LIM);
    }
    scan2(cn, ct, &tn, &tt, red);
    unsigned fits = 0;
    int total = 0, blocks = 0;   // tokens and blocks of the sequences that fit
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (s0 + i >= n) continue;
        first[s0 + i] = (int)cn; start[s0 + i] = (int)ct;
        cn = min(cn + need[i], (unsigned)KP_LIM); ct = min(ct + tok[i], (unsigned)KP_LIM);
        if (cn <= (unsigned)nfree && ct <= (unsigned)a.ntok && ct < KP_LIM) { fits |= 1u << i; total = (int)ct; blocks = (int)cn; }
    }
    // sums only grow: the largest of those that fit are the totals
    total = wave_max(total); blocks = wave_max(blocks);
    __syncthreads();   // red has been read
    if ((tid & 63) == 0) red[tid >> 6] = make_uint2(total, blocks);
    __syncthreads();
    for (int i = 0; i < nt >> 6; i++) { total = max(total, (int)red[i].x); blocks = max(blocks, (int)red[i].y); }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (s0 + i >= n) continue;
        if (!((fits >> i) & 1)) { start[s0 + i] = total; first[s0 + i] = blocks; add[i] = 0; }
        a.qstart[s0 + i] = start[s0 + i];
        a.len[s0 + i] = lens[s0 + i] = ctx[i] + add[i];
    }
    if (tid == 0) { start[n] = total; first[n] = blocks; a.qstart[n] = total; a.nfree_out[0] = nfree - blocks; }
    __syncthreads();
    // 3. new blocks, from the end of the list; then the tokens
    for (int j = tid; j < blocks; j += nt) {
        int s = count_le(first, n, j) - 1;
        int held = (lens[s] - (start[s + 1] - start[s]) + bs1) >> sh;
        a.table[(int64_t)s * a.width + held + j - first[s]] = taken(j);
    }
    if (!tokens) return;
    for (int t = tid; t < a.ntok; t += nt) {
        int pos = 0, slot = -1;
        if (t < total) {
            const int s = count_le(start, n, t) - 1, c = lens[s] - (start[s + 1] - start[s]);
            pos = c + t - start[s];
            const int j = (pos >> sh) - ((c + bs1) >> sh) + first[s];   // of the blocks taken; before the sequence's first: the begun one
            const int blk = j < first[s] ? tail[s] : taken(j);
            if ((unsigned)blk < (unsigned)a.nblocks) slot = (blk << sh) + (pos & bs1);
        }
        a.pos[t] = pos; a.slot[t] = slot;
    }
}

// The tokens of a large step, in a launch of their own over the whole card: 60000 in 2.7 us (their starts into LDS, then a search and two
// dependent loads; 0.5 MB written)
__global__ void __launch_bounds__(256) k_kv_tokens(mmoe_kv_plan_args a, int sh) {
    __shared__ int start[MMOE_KV_MAXSEQ + 1];
    for (int i = threadIdx.x; i <= a.nseq; i += 256) start[i] = a.qstart[i];
    __syncthreads();
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.ntok) return;
    int pos = 0, slot = -1;
    if (t < start[a.nseq]) {
        const int s = count_le(start, a.nseq, t) - 1;
        pos = a.len[s] - (start[s + 1] - t);
        const int blk = a.table[(int64_t)s * a.width + (pos >> sh)];
        if ((unsigned)blk < (unsigned)a.nblocks) slot = (blk << sh) + (pos & (a.block_size - 1));
    }
    a.pos[t] = pos; a.slot[t] = slot;
}

// ------------------------------------------------------------------------------------------------------
// Rotary positions and the cache write (mmoe_rope_kv)
// ------------------------------------------------------------------------------------------------------
// A workgroup takes tb tokens: their cos / sin into LDS once for all heads, then the heads in units of 8 values. The angle is
// reduced to half turns in 64 bits (pos * freq reaches 1e6 radians, where 32 bits are 0.06 off) before the 32-bit sine. Bound by the
// bytes at long prompts (8191 tokens of 24 heads of 128 in bf16: 100.7 MB in 22.9 us, 4.4 TB/s; a copy of as many reaches 4.9), by latency
// at short ones (64 tokens 3.8 us, 777 tokens 4.8 us: the angles' 64-bit product and sine beside the first heads' loads).
#define RP_T 256
#define RP_HALF 128   // largest rot / 2
#define RP_TB 8       // most tokens per workgroup
#define RP_U 3        // heads of a lane whose loads are under way together (8191 tokens: 1 or 2 26.5 us, 3 24.1, 4 26.5, 6 26.0: with 3 two tokens of
                      // Maple's 24 heads are one turn)
enum { RP_INTER, RP_SPLIT, RP_ODD };   // pairs (2 i, 2 i + 1); (i, i + rot / 2) with rot / 2 in whole units of 8; any rot, any head_dim

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

// Head hd of a token's query heads | key heads | value heads (the last with a cache only): where it comes from and goes to (NULL: nowhere).
struct RopeHead {
    const void *in;
    int64_t src;
    uint8_t *out;
    bool turn;
};
template <int OUT> __device__ __forceinline__ RopeHead rope_head(const mmoe_rope_args &a, const mmoe_kv_cache &kv, int cached, int sh, int64_t tok, int hd) {
    RopeHead r;
    bool live = true;
    int64_t slot = 0, dst;
    void *out;
    if (cached) {
        int s = a.slot[tok];
        live = s >= 0 && (s >> sh) < kv.nblocks;
        slot = (int64_t)(s >> sh) * kv.block_stride + (int64_t)(s & (kv.block_size - 1)) * kv.token_stride;
    }
    int hk = hd - a.heads, hv = hk - a.kv_heads;
    r.turn = hv < 0;
    if (hk < 0) { r.in = a.q; r.src = tok * a.q_token + hd * a.q_head; out = a.q_out; dst = tok * a.qo_token + hd * a.qo_head; }
    else if (hv < 0) {
        r.in = a.k; r.src = tok * a.k_token + hk * a.k_head;
        out = cached ? kv.k : a.k_out;
        dst = cached ? slot + hk * kv.head_stride : tok * a.ko_token + hk * a.ko_head;
    } else { r.in = a.v; r.src = tok * a.v_token + hv * a.v_head; out = kv.v; dst = slot + hv * kv.head_stride; }
    r.out = live ? (uint8_t *)out + dst * Elem<OUT>::size : nullptr;
    return r;
}

template <int IN, int OUT, int LAY>
__global__ void __launch_bounds__(RP_T) k_rope(mmoe_rope_args a, mmoe_kv_cache kv, int cached, int sh, int tb) {
    __shared__ float2 cs[RP_TB * RP_HALF];
    __shared__ float row[LAY == RP_ODD ? RP_T * 8 : 1];
    const int t0 = blockIdx.x * tb, nt = min(tb, a.ntok - t0), half = a.rot >> 1, dc = a.head_dim >> 3;
    const int nh = a.heads + a.kv_heads + (cached ? a.kv_heads : 0), all = nt * nh;   // heads of the workgroup's tokens
    if (LAY == RP_ODD) {
        rope_angles(a, t0, nt, cs);
        __syncthreads();
        // the round's heads through LDS: a unit's partners start anywhere in another unit. Two barriers a round and no loads ahead: 8191 tokens of
        // Maple's heads with rot 20 in 29 us, with rot 64 (split) 23; 64 tokens cost the same
        const int hpr = RP_T / dc, hl = threadIdx.x / dc, d0 = (threadIdx.x - hl * dc) * 8;
        for (int j0 = 0; j0 < all; j0 += hpr) {
            int j = j0 + hl, t = j / nh;
            bool on = hl < hpr && j < all;
            RopeHead r;
            float x[8], y[8], *mine = row + threadIdx.x * 8, *head = row + hl * a.head_dim;
            if (on) {
                r = rope_head<OUT>(a, kv, cached, sh, t0 + t, j - t * nh);
                on = r.out != nullptr;
            }
            if (on) {
                unpack8<IN>(x, load8<IN>(r.in, r.src + d0));
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
                    const bool low = a.interleaved ? !(d & 1) : d < half;   // of its pair
                    const float2 c = cs[t * RP_HALF + (a.interleaved ? d >> 1 : low ? d : d - half)];
                    const float z = head[a.interleaved ? d ^ 1 : low ? d + half : d - half];
                    y[i] = low ? fmaf(x[i], c.x, -(z * c.y)) : fmaf(x[i], c.x, z * c.y);
                }
                store8<OUT>(r.out + d0 * Elem<OUT>::size, y);
            }
            __syncthreads();
        }
        return;
    }
    // A head is dc lanes of one wave (dc a power of two), a unit of 8 values each; RP_U heads' loads under way per lane, the first ones
    // beside the angles. With split pairs a lane loads its partner's unit too (the same lines again): in place, too, a head is read
    // whole before any of it is written.
    const int sd = 31 - __builtin_clz(dc), d0 = (threadIdx.x & (dc - 1)) * 8, hpr = RP_T >> sd;
    int hd = threadIdx.x >> sd, t = 0;
    Raw8<IN> x[RP_U], z[RP_U];
    uint8_t *out[RP_U];
    int tk[RP_U];
    bool turn[RP_U];
    auto load = [&](int left) {
#pragma unroll
        for (int k = 0; k < RP_U; k++) {
            out[k] = nullptr;
            if (k >= left) continue;
            while (hd >= nh) { hd -= nh; t++; }
            const RopeHead r = rope_head<OUT>(a, kv, cached, sh, t0 + t, hd);
            out[k] = r.out ? r.out + d0 * Elem<OUT>::size : nullptr;
            turn[k] = r.turn && d0 < a.rot;
            tk[k] = t;
            hd += hpr;
            x[k] = load8<IN>(r.in, r.src + d0);
            if (LAY == RP_SPLIT && turn[k]) z[k] = load8<IN>(r.in, r.src + (d0 < half ? d0 + half : d0 - half));
        }
    };
    auto store = [&] {
#pragma unroll
        for (int k = 0; k < RP_U; k++) {
            if (!out[k]) continue;
            float y[8];
            unpack8<IN>(y, x[k]);
            if (turn[k]) {
                const float2 *w = cs + tk[k] * RP_HALF;
                if (LAY == RP_INTER) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        if (d0 + i >= a.rot) continue;
                        const float2 c = w[(d0 + i) >> 1];
                        const float lo = y[i], hi = y[i + 1];
                        y[i] = fmaf(lo, c.x, -(hi * c.y));
                        y[i + 1] = fmaf(hi, c.x, lo * c.y);
                    }
                } else {
                    float other[8];
                    unpack8<IN>(other, z[k]);
                    const float sign = d0 < half ? -1.0f : 1.0f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float2 c = w[(d0 < half ? d0 : d0 - half) + i];
                        y[i] = fmaf(y[i], c.x, sign * (other[i] * c.y));
                    }
                }
            }
            store8<OUT>(out[k], y);
        }
    };
    int left = (all - hd + hpr - 1) / hpr;
    load(left);
    rope_angles(a, t0, nt, cs);
    __syncthreads();
    for (;;) {
        store();
        if ((left -= RP_U) <= 0) return;
        load(left);
    }
}

// ------------------------------------------------------------------------------------------------------
// Attention over the blocks (mmoe_attn_paged)
// ------------------------------------------------------------------------------------------------------
// Every kernel here keeps a softmax's running maximum and sum and one pass over the positions. A query row is a (token, query
// head) pair; the rows that read one key/value head, token by token and its group of query heads within, share its keys. The
// rows' visible runs [lo, hi) are all there is to masks: a tile that every live row sees whole needs none.
#define ATT_BM 128         // rows of a tile
#define ATT_BN(D) (8192 / (D))   // and its positions: 32 KB of keys and values for either head size
#define ATT_LOG2E 1.44269504088896340736f
#define ATT_LN2 0.69314718055994530942f

typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s4v ls4;
typedef __attribute__((address_space(3))) u4 lu4;
typedef __attribute__((address_space(3))) uint8_t lb;
typedef __attribute__((address_space(1))) const uint8_t gb;

// n / d for every 32-bit n by a multiplication (Granlund and Montgomery 1994); a division costs some 40 instructions
struct Div {
    uint32_t d, m, s1, s2;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { uint32_t t = __umulhi(m, n); return (t + ((n - t) >> s1)) >> s2; }
};

struct AttArgs {
    mmoe_attn_args a;
    mmoe_kv_cache kv;
    int sh, group;       // log2 of the block size, query heads per key/value head
    Div by_heads, by_kv, by_group, by_split, by_split_sh, by_chunks;
    // one launch: n_sh workgroups over the shared positions (row tiles of 128, or of 16 with sh_few), n_tile over each sequence's own
    // positions in row tiles of 128, n_few over those of sequences with up to `few` rows per key/value head (0: none) in chunks
    unsigned n_sh, n_tile, n_few;
    int tiles_sh, tiles;   // their row tiles
    int sh_few, few;
    int split_sh, split, chunk, chunks;   // runs of the shared positions, runs per row tile of the own ones; positions per chunk, most chunks
    int parts_sh;        // partial results of the shared positions: split_sh, or 0
    float s1, s2;        // cap 0: score = s1 q.k in units of log 2; else s2 tanh z, with exp(2 z) = exp2(s1 q.k)
    // partial results, [head_dim] values over their own sum each, and their maxima (in units of log 2) and sums (negative where results may not
    // be finite): of the shared positions
    // [split_sh][ntok][heads], from at_tile on of row tiles over the own ones [split][ntok][heads], from at_few on of chunks [chunks][nseq][16 kv heads]
    float *po;
    float2 *pm;
    int64_t at_tile, at_few;
};

template <int T> __device__ __forceinline__ f16v mfma32(u4 a, u4 b, f16v c) {
    if (T == MMOE_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
// Weights are 2^(x - m + lift): in fp16 their smallest step is 2^-24, which a tail of many small weights would be rounded to; lifted by 2^7
// (they reach 2^15 before the maximum m follows) it is 2^-31 of the largest weight. Sums and results carry the same factor.
// Past 2^20 a maximum takes no lift (m - lift would be rounded), and scores are rounded before it is subtracted: a fused multiply-add's own,
// more exact one may lie half a step of m above it, and at 2^24 that is a factor of 2 in the weight.
template <int T> constexpr float lift = T == MMOE_F16 ? 7.0f : 0.0f;
#define ATT_FAR 1048576.0f
template <int T> __device__ __forceinline__ float lowered(float m) { return fabsf(m) > ATT_FAR ? m : m - lift<T>; }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// the larger of two numbers, without fmaxf's quieting of each (a NaN shows in the weights, whatever the maximum then is)
__device__ __forceinline__ float max_(float x, float y) { return __builtin_amdgcn_fmed3f(x, y, __builtin_inff()); }
__device__ __forceinline__ float min_(float x, float y) { return __builtin_amdgcn_fmed3f(x, y, -__builtin_inff()); }
// N pieces of 16 bytes per lane from base + off[i] + 1024 i to LDS at to + 1024 i + 16 * lane (the offset of the instruction counts on both
// sides). Asm, so that the compiler does not wait for them before every later LDS read; nothing is written to a register. The
// waits are the caller's.
template <int N> __device__ __forceinline__ void load_lds(const uint8_t *base, const uint32_t *off, uint32_t to) {
    static_assert(N == 2 || N == 4, "loads");
    to = __builtin_amdgcn_readfirstlane(to);
    if (N == 2)
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x400" ::"v"(off[0]), "v"(off[1]), "s"(base), "s"(to)
                     : "memory", "m0");
    if (N == 4)
        asm volatile("s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\tglobal_load_lds_dwordx4 %1, %4 offset:0x400\n\t"
                     "global_load_lds_dwordx4 %2, %4 offset:0x800\n\tglobal_load_lds_dwordx4 %3, %4 offset:0xc00" ::"v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(to)
                     : "memory", "m0");
}
// what two half-waves hold of one column
__device__ __forceinline__ float max_halves(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The sequence and row tile of virtual tile v, with tiles of bm rows: sequence s has the tiles from floor(rows before it / bm) + s
// on; no two sequences' tiles meet, and some virtual tiles are nobody's. No sums over the sequences are needed.
__device__ __forceinline__ int att_start(const mmoe_attn_args &a, int s) { return min(max(a.qstart[s], 0), a.ntok); }   // never past the arrays
struct AttTileAt { int s, row0, rows, t0; };   // first row of the tile in its sequence, the sequence's rows, its first token
__device__ __forceinline__ bool att_find(const AttArgs &A, bool shared, int bm, int v, AttTileAt &o) {
    const mmoe_attn_args &a = A.a;
    if (shared) {
        o.s = 0; o.t0 = 0; o.row0 = v * bm; o.rows = att_start(a, a.nseq) * A.group;
        return o.row0 < o.rows;
    }
    // the last s whose first tile is <= v
    const int lo = a.nseq == 1 ? 0 : max(count_wave(a.nseq, [&](int m) { return (int)((int64_t)att_start(a, m) * A.group / bm) + m <= v; }) - 1, 0);
    o.s = lo; o.t0 = att_start(a, lo);
    o.row0 = (v - (int)((int64_t)o.t0 * A.group / bm) - lo) * bm;
    o.rows = min(att_start(a, lo + 1) - o.t0, a.max_q) * A.group;
    return o.row0 < o.rows && o.rows > A.few;
}
// A sequence's own positions `from` .. `to` in chunks, n of them, at least one (att_few and k_attn_join agree through this)
struct AttChunks { int from, n, to; };
__device__ __forceinline__ AttChunks att_chunks(const AttArgs &A, int s, int tokens) {
    const mmoe_attn_args &a = A.a;
    int len = a.len[s], from = a.shared, to = a.hi ? len : len - max(tokens - a.max_q, 0);   // the last served token's end
    if (a.window > 0) from = max(from, len - tokens - a.window);
    from &= ~31;
    to = min(to, a.max_len);
    return {from, to > from ? min((to - from + A.chunk - 1) / A.chunk, A.chunks) : 1, to};
}

// One query row as a lane sees it: its token and head, then (with a search for its sequence, if that is not the tile's) its limits
struct AttRow { int tok, head, pos, lo, hi; bool live; };
__device__ __forceinline__ AttRow att_row(const AttArgs &A, const AttTileAt &at, int r, int kvh) {
    AttRow o;
    o.live = r < at.rows;
    if (!o.live) r = at.rows - 1;
    const int j = (int)A.by_group(r);
    o.tok = at.t0 + j;
    o.head = kvh * A.group + r - j * A.group;
    return o;
}
// Its sequence. starts: room for all of qstart in LDS, every thread of the workgroup here
struct AttSeq { int s, t0, t1; };
__device__ __forceinline__ AttSeq att_seq(const AttArgs &A, bool shared, const AttTileAt &at, int *starts, const AttRow &o) {
    const mmoe_attn_args &a = A.a;
    int s = at.s, t0, t1;
    if (shared) {
        for (int i = threadIdx.x; i <= a.nseq; i += blockDim.x) starts[i] = a.qstart[i];
        __syncthreads();
        s = max(count_le(starts, a.nseq, o.tok) - 1, 0);
        t0 = starts[s]; t1 = starts[s + 1];
        __syncthreads();
    } else { t0 = a.qstart[s]; t1 = a.qstart[s + 1]; }
    return {s, t0, t1};
}
__device__ __forceinline__ void att_limits(const AttArgs &A, bool shared, const AttSeq &q, AttRow &o) {
    const mmoe_attn_args &a = A.a;
    int len = a.len[q.s];
    o.pos = len - (q.t1 - o.tok);
    if (o.tok - q.t0 >= a.max_q) o.live = false;
    o.lo = a.lo ? max(a.lo[o.tok], 0) : 0;
    o.hi = a.hi ? a.hi[o.tok] : o.pos + 1;
    if (a.window > 0) o.lo = max(o.lo, o.pos - a.window);
    o.hi = max(min(min(o.hi, len), a.max_len), 0);
    if (shared) o.hi = min(o.hi, a.shared); else o.lo = max(o.lo, a.shared);
}

// Values of a tile that is not seen whole: are all of them finite? (bits: the type's exponent)
template <int T> __device__ __forceinline__ bool odd16(uint32_t v) { constexpr uint32_t e = T == MMOE_BF16 ? 0x7f80 : 0x7c00; return (v & e) == e; }
// the same of both halves of a word: bit 15 or 31 set (a carry out of the exponent; other bits are of no meaning)
template <int T> __device__ __forceinline__ uint32_t odd_pair(uint32_t v) { return (v & 0x7fff7fffu) + (T == MMOE_BF16 ? 0x00800080u : 0x04000400u); }
// what is left of a result whose weight has become 0
__device__ __forceinline__ float only_odd(float y) { return __builtin_isfinite(y) ? 0.0f : y; }
// the largest size of two numbers, NaN if one of them is
__device__ __forceinline__ float largest_of(float x, float y) { return __builtin_elementwise_maximum(fabsf(x), fabsf(y)); }
template <int T> __device__ __forceinline__ uint32_t only_finite(uint32_t v) {
    if (odd16<T>(v)) v &= 0xffff0000u;
    if (odd16<T>(v >> 16)) v &= 0xffffu;
    return v;
}

// Row tiles of 4 waves, 32 rows each, over tiles of 64 positions (128 with heads of 64) that all waves share through LDS.
// S^T = K Q^T, so a lane holds one row's scores (half of the positions, the other half in the lane 32 away): the softmax needs
// one exchange per tile, and P^T, packed to 16 bits, is the second product's operand as it lies. O^T = V^T P^T takes its V^T from
// rows of V through the transposing LDS reads. A tile's keys and values go from the cache straight to LDS, one tile ahead, in 16-byte
// pieces whose place in a row is exchanged by the row's number, so that neither the reads of 8 rows at one column nor the transposing
// reads of 4 rows meet in a bank. P is rounded to the cache's type (half a step relative, as the result itself is), its
// sum is of the unrounded 32-bit values. With two workgroups on a CU a SIMD's two waves take turns: one's matrix products (which go
// first, s_setprio: 6% of a long run) run beside the other's exponentials.
// Bound at long runs: 4096 tokens over 16096 positions, 16 heads of 128, 471 GFLOP: 451 to 472 us on several cards, 1.0 PFLOP/s (a product of
// 8192 cubed reaches 1.28; the clock falls to 1.5 GHz); with a cap 530 to 553 (three more instructions and two of the transcendental unit per
// score), with a distance bias 510 to 533. Short runs: 2.5 us to the first tile (sequence, limits, block ids, tile: loads that depend on each
// other), 1.7 us per tile of a wave alone on its SIMD.
template <int D> struct AttTileMem {
    __attribute__((aligned(1024))) uint8_t first[2 * ATT_BN(D) * D * 2];   // keys and values of a tile
    union {
        __attribute__((aligned(1024))) uint8_t second[2 * ATT_BN(D) * D * 2];
        int starts[MMOE_KV_MAXSEQ + 1];
    };
    int range[4][4], flag[2][4];
};
template <int T, int D, bool CAP, bool BIAS>
__device__ __forceinline__ void att_tile(const AttArgs &A, const bool shared, const unsigned block, AttTileMem<D> &M) {
    constexpr int RB = D * 2, CH = D / 8, RPI = 64 / CH, NI = 16 / RPI, KS = D / 16, DS = D / 32;   // a row's bytes and chunks; rows of a load, loads of 16 rows
    constexpr int BN = ATT_BN(D), GW = BN / 64, NU = BN / 32, NK = BN / 16;   // groups of 16 positions that a wave loads; score blocks, steps of the second product
    constexpr uint32_t TB = BN * RB;
    const mmoe_attn_args &a = A.a;
    const int nsplit = shared ? A.split_sh : A.split;
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = l & 31, hh = l >> 5;
    const unsigned rest = A.by_kv(block), v = (shared ? A.by_split_sh : A.by_split)(rest);
    const int kvh = block - rest * A.kv.heads, split = rest - v * nsplit;
    AttTileAt at;
    // a sequence's last tiles see most: first (the sequences in reverse order, whatever their lengths)
    if (!att_find(A, shared, ATT_BM, (shared ? A.tiles_sh : A.tiles) - 1 - (int)v, at)) return;

    // What the lane loads of a tile: row RPI i + l / CH of the wave's 16, piece l % CH of LDS, less the instruction's own offset (rows are at
    // least head_dim values apart, so it stays positive).
    uint32_t ko[NI], vo[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        int r = RPI * i + l / CH, c = l % CH;
        ko[i] = (uint32_t)(r * A.kv.token_stride + (c ^ (r & (CH - 1))) * 8) * 2 - 1024 * i;
        vo[i] = (uint32_t)(r * A.kv.token_stride + (c ^ ((r & (CH / 2 - 1)) << 1)) * 8) * 2 - 1024 * i;
    }
    // block ids of 64 groups of 16 positions at a time, group l in lane l; a load of their own each tile would have to be waited for
    // with the tile's
    const int32_t *table = a.table + (int64_t)at.s * a.width;
    int id = 0, idp = INT32_MIN / 2;      // ids of the positions from idp on
    uint64_t lost = 0;                    // those that are none of the cache's
    auto block_of = [&](int p, unsigned &bad) {   // the wave's blocks of a tile
        if (p - idp >= 1024) {
            idp = p;
            id = table[min((p + 16 * l) >> A.sh, a.width - 1)];
            lost = __ballot((unsigned)id >= (unsigned)A.kv.nblocks);
        }
        bad = (unsigned)(lost >> ((p - idp) >> 4)) & ((1u << NK) - 1);
        struct { int at[GW]; } blk;
#pragma unroll
        for (int g = 0; g < GW; g++) {
            const int b = __builtin_amdgcn_readlane(id, ((p - idp) >> 4) + GW * w + g);
            blk.at[g] = (unsigned)b < (unsigned)A.kv.nblocks ? b : 0;
        }
        return blk;
    };
    auto fetch = [&](uint32_t buf, const void *base, const uint32_t *off, int p, const auto &blk) {
#pragma unroll
        for (int g = 0; g < GW; g++) {
            const int r = 16 * (GW * w + g);
            const uint8_t *from = (const uint8_t *)base + (blk.at[g] * A.kv.block_stride + kvh * A.kv.head_stride + ((p + r) & (A.kv.block_size - 1)) * A.kv.token_stride) * 2;
            load_lds<NI>(from, off, buf + r * RB);
        }
    };
    const uint32_t lds = (uint32_t)(uintptr_t)(lb *)M.first;   // tile i: keys at lds + 2 TB (i % 2), values TB behind them
    unsigned bad = 0, next = 0;   // the tile's lost blocks, the next one's
    int p0, p1;
    decltype(block_of(0, bad)) blk;
    if (shared) {   // which positions is known already: the first tile comes while the rows look for their sequences
        const int run = ((a.shared + BN - 1) / BN + nsplit - 1) / nsplit * BN;
        p0 = split * run; p1 = min(p0 + run, a.shared);
        if (p0 < p1) {
            blk = block_of(p0, bad);
            fetch(lds, A.kv.k, ko, p0, blk);
            fetch(lds + TB, A.kv.v, vo, p0, blk);
        }
    }
    AttRow R = att_row(A, at, at.row0 + w * 32 + n, kvh);
    att_limits(A, shared, att_seq(A, shared, at, M.starts, R), R);
    // queries: operand B, lane (hh, n) holds dims 16 s + 8 hh .. + 8 of row n
    u4 q[KS];
    {
        const uint16_t *qp = (const uint16_t *)a.q + (int64_t)R.tok * a.q_token + R.head * a.q_head + 8 * hh;
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = *(const gu4 *)(qp + 16 * s);
    }
    // A score is sc s1 + s0 in units of log 2, in which sc is the product's with the bias in its units, or with a cap 1 / (1 + exp 2 z):
    // what is left of them is in the exponentials' own multiplication.
    const float s0 = CAP && !BIAS ? A.s2 : 0.0f, s1 = CAP ? BIAS ? 1.0f : -2.0f * A.s2 : A.s1;
    const float slope = BIAS ? a.slopes[R.head] * (CAP ? ATT_LOG2E : ATT_LOG2E / A.s1) : 0.0f;
    // the wave's and the workgroup's positions
    const bool some = R.live && R.lo < R.hi;
    const int wlo = wave_min(some ? R.lo : INT32_MAX), whi = wave_max(some ? R.hi : 0);
    const int inlo = wave_max(R.live ? R.lo : 0), inhi = wave_min(R.live ? R.hi : INT32_MAX);
    if (l == 0) { M.range[0][w] = wlo; M.range[1][w] = whi; M.range[2][w] = inlo; M.range[3][w] = inhi; }
    __syncthreads();
    int lo = INT32_MAX, hi = 0, glo = 0, ghi = INT32_MAX;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        lo = min(lo, M.range[0][i]); hi = max(hi, M.range[1][i]);
        glo = max(glo, M.range[2][i]); ghi = min(ghi, M.range[3][i]);
    }
    const int seen = __builtin_amdgcn_readfirstlane(lo);   // the first position that any row sees
    lo = seen & ~(BN - 1); hi = __builtin_amdgcn_readfirstlane(hi);
    glo = __builtin_amdgcn_readfirstlane(glo); ghi = __builtin_amdgcn_readfirstlane(ghi);
    if (shared) {
        p1 = lo < hi ? min(p1, hi) : p0;   // (the first tile is there, also where it lies before lo: nobody looks)
        if (p0 >= p1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // and is not left on its way into LDS that is another's
    } else {
        p0 = lo; p1 = hi;
        if (nsplit > 1 && p0 < p1) {
            int run = ((p1 - p0 + BN - 1) / BN + nsplit - 1) / nsplit * BN;
            p0 += split * run;
            p1 = min(p1, p0 + run);
        }
        if (p0 < p1) {
            blk = block_of(p0, bad);
            fetch(lds, A.kv.k, ko, p0, blk);
            fetch(lds + TB, A.kv.v, vo, p0, blk);
        }
    }
    // where it reads them back: K row n (and n + 32), pieces 2 k + hh; V rows vr (and on by eights), dims 32 i + 16 (l / 16 % 2) + 4 (l % 4) ..
    // (the number that exchanges a row's pieces is the same for rows 32 (K) and 8 (V) apart: what is added are constants)
    uint32_t ka[KS], va[DS];
    const int vr = 4 * hh + ((l & 15) >> 2);
#pragma unroll
    for (int k = 0; k < KS; k++) ka[k] = n * RB + (((2 * k + hh) ^ (n & (CH - 1))) << 4);
#pragma unroll
    for (int i = 0; i < DS; i++) va[i] = vr * RB + ((64 * i + 32 * ((l >> 4) & 1) + 8 * (l & 3)) ^ ((vr & (CH / 2 - 1)) << 5));
    f16v acc[DS], sc[NU];
    float m, mb, sum;   // mb: m - lift, - lift while m is -inf
    bool far;           // a maximum of the wave is past ATT_FAR
    constexpr bool FALLS = CAP && !BIAS;   // sc falls as the score grows
    constexpr float NONE = FALLS ? __builtin_inff() : -__builtin_inff();   // sc of a position that is not seen

    auto scores = [&](f16v *s, uint32_t buf) {
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[u][j] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int u = 0; u < NU; u++) s[u] = mfma32<T>(*(const lu4 *)((const lb *)(uintptr_t)buf + ka[k] + 32 * u * RB), q[k], s[u]);
        // six reads ahead of the products
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int k = 0; k < NU * KS - 6; k++) { __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); }
        __builtin_amdgcn_sched_group_barrier(0x8, 6, 0);
    };
    auto math = [&](f16v *s, int p) {
        const float dist = BIAS ? (float)(R.pos - p - 4 * hh) : 0.0f;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                float x = s[u][j];
                if (CAP) x = __builtin_amdgcn_rcpf(1.0f + exp2_(x * A.s1));   // tanh z = 1 - 2 / (1 + exp 2 z)
                if (CAP && BIAS) x = fmaf(-2.0f * A.s2, x, A.s2);
                if (BIAS) x = fmaf(-slope, fabsf(dist - (float)(32 * u + 8 * (j >> 2) + (j & 3))), x);
                s[u][j] = x;
            }
    };
    // a tile that is not seen whole: a score of -inf where a row does not look
    auto mask = [&](f16v *s, int p, unsigned bad) {
        const unsigned at = (unsigned)(p + 4 * hh - R.lo), span = (unsigned)max(R.hi - R.lo, 0);
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[u][j] = at + (32 * u + 8 * (j >> 2) + (j & 3)) < span ? s[u][j] : NONE;
        if (bad)
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int j = 0; j < 16; j++) s[u][j] = (bad >> (2 * u + (j >> 3))) & 1 ? NONE : s[u][j];
    };
    auto largest = [&](const f16v *s) {
        float top[4];   // no chain of 32
        auto higher = [](float x, float y) { return FALLS ? min_(x, y) : max_(x, y); };
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < 16; j++) top[j & 3] = u || j > 3 ? higher(top[j & 3], s[u][j]) : s[u][j];
        return max_halves(fmaf(higher(higher(top[0], top[1]), higher(top[2], top[3])), s1, s0));
    };
    // a new maximum only once it is 2^8 past the old: until then weights stay below 2^8 (lifted: 2^15), in every type's range
    auto rescale = [&](float mt) {
        if (!__any(mt - m > 8.0f)) return;
        const float mn = fmaxf(m, mt), bn = lowered<T>(mn == -__builtin_inff() ? 0.0f : mn), al = m == -__builtin_inff() ? 0.0f : exp2_(mb - bn);
        m = mn; mb = bn; sum *= al;
        far = __any(fabsf(bn) > ATT_FAR);
#pragma unroll
        for (int i = 0; i < DS; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) acc[i][j] *= al;
    };
    auto product = [&](uint32_t vbuf) {
        // V^T: lane (hh, n) of operand A holds dim 32 i + n, positions 16 k + 4 hh + {0 .. 3, 8 .. 11}
        auto value = [&](int i, int k) {
            const lb *v = (const lb *)(uintptr_t)vbuf + va[i] + 16 * k * RB;
            uint2 t0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)v));
            uint2 t1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)(v + 8 * RB)));
            return u4{t0.x, t0.y, t1.x, t1.y};
        };
        constexpr int AHEAD = 4 / DS;
        u4 f0[4];   // the first positions' are on their way during the exponentials
#pragma unroll
        for (int i = 0; i < 4; i++) f0[i] = value(i % DS, i / DS);
        __builtin_amdgcn_sched_barrier(0);
        u4 pf[NK];
        float part = 0;
        const float mul = far ? 1.0f : s1, off = far ? -mb : s0 - mb;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                float e0 = exp2_(fmaf(sc[u][j], mul, off)), e1 = exp2_(fmaf(sc[u][j + 1], mul, off));
                part += e0 + e1;
                pf[2 * u + (j >> 3)][(j & 7) >> 1] = pack2<T>(e0, e1);
            }
        sum += part;   // tile by tile: a long sum of small ones
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int i = 0; i < DS; i++) acc[i] = mfma32<T>(k < AHEAD ? f0[k * DS + i] : value(i, k), pf[k], acc[i]);
#pragma unroll
        for (int k = 0; k < NK * DS - 4; k++) { __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
    };
    // A value that is not finite times a weight of 0 is NaN, so in a tile that is not seen whole such values are zeroed before the product
    // and, once all tiles are through, added as they are to the rows that see their position. In a tile seen whole the product is right unless
    // a small weight was rounded to 0, or later scaled to 0: then the result is NaN, and the row tile begins again with every tile's
    // values looked at (at once, that would be an eighth more reads of LDS for every call).
    // the wave's own rows of values: 1 if some are not finite, 2 if a row of the tile may see one
    auto look = [&](uint32_t buf, int p, int f) {
        uint32_t o = 0, see = 0;
#pragma unroll
        for (int x = 0; x < GW * NI; x++) {
            u4 v = *(const lu4 *)((const lb *)(uintptr_t)buf + w * 16 * GW * RB + x * 1024 + l * 16);
            uint32_t mine = 0;
#pragma unroll
            for (int y = 0; y < 4; y++) mine |= odd_pair<T>(v[y]);
            const int at = p + w * 16 * GW + x * RPI + l / CH;
            o |= mine;
            see |= at >= seen && at < hi ? mine : 0;
        }
        const int bits = (__any((o & 0x80008000u) != 0) ? 1 : 0) | (__any((see & 0x80008000u) != 0) ? 2 : 0);
        if (l == 0) M.flag[f][w] = bits;
    };
    auto found = [&](int f) { return __builtin_amdgcn_readfirstlane(M.flag[f][0] | M.flag[f][1] | M.flag[f][2] | M.flag[f][3]); };
    auto zero_odd = [&](uint32_t buf) {
#pragma unroll
        for (int x = 0; x < GW * NI; x++) {
            lu4 *at = (lu4 *)((lb *)(uintptr_t)buf + w * 16 * GW * RB + x * 1024 + l * 16);
            u4 v = *at;
#pragma unroll
            for (int y = 0; y < 4; y++) v[y] = only_finite<T>(v[y]);
            *at = v;
        }
    };
    auto add_odd = [&](uint32_t buf, int p, unsigned bad) {
#pragma unroll 1
        for (int r = 0; r < BN; r++) {
            const bool see = p + r >= R.lo && p + r < R.hi && !((bad >> (r >> 4)) & 1);
            uint32_t row = r * RB + 8 * hh, x = (r & (CH / 2 - 1)) << 5;
            asm("" : "+v"(row));   // its addresses are not worth a register outside
#pragma unroll
            for (int i = 0; i < DS; i++)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    typedef __attribute__((address_space(3))) uint64_t l8;
                    uint64_t v = *(const l8 *)((const lb *)(uintptr_t)buf + row + ((64 * i + 4 * j) ^ x));
#pragma unroll
                    for (int y = 0; y < 4; y++, v >>= 16) {
                        acc[i][j + y] += see && odd16<T>((uint32_t)v) ? half_to_f<T>((uint32_t)v & 0xffff) : 0.0f;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
        }
    };

#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(q[s]));   // the queries are there, on every way into the loop: nothing in it waits for them
    int odd0 = INT32_MAX, odd1 = 0;   // the tiles in which some row may see a value that was zeroed
    bool wild = false;                // results of the wave may not be finite
    for (bool careful = false;; careful = true) {
        m = -__builtin_inff(); mb = sum = 0.0f; far = false;
#pragma unroll
        for (int i = 0; i < DS; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) acc[i][j] = 0.0f;
        for (int p = p0, i = 0; p < p1; p += BN, i ^= 1, bad = next) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the compiler does not know of these loads
            const uint32_t kbuf = lds + i * 2 * TB, vbuf = kbuf + TB, kother = lds + (i ^ 1) * 2 * TB;
            const bool part = careful || p < glo || p + BN > ghi || bad;
            if (part) look(vbuf, p, i);
            __syncthreads();   // the tile has arrived, and every wave is done with the other buffers
            if (p + BN < p1) {
                blk = block_of(p + BN, next);
                fetch(kother, A.kv.k, ko, p + BN, blk);
                fetch(kother + TB, A.kv.v, vo, p + BN, blk);
            }
            const int odd = part ? found(i) : 0;
            if (odd) {
                if (odd & 2) { odd0 = min(odd0, p); odd1 = p + 1; }
                zero_odd(vbuf);
                __syncthreads();
            }
            if (p < whi && p + BN > wlo) {
                __builtin_amdgcn_s_setprio(1);
                scores(sc, kbuf);
                __builtin_amdgcn_s_setprio(0);
                if (CAP || BIAS) math(sc, p);
                if (p < inlo || p + BN > inhi || bad) mask(sc, p, bad);
                rescale(largest(sc));
                if (far) {
#pragma unroll
                    for (int u = 0; u < NU; u++)
#pragma unroll
                        for (int j = 0; j < 16; j++) sc[u][j] = fmaf(sc[u][j], s1, s0);
                }
                __builtin_amdgcn_s_setprio(1);
                product(vbuf);
                __builtin_amdgcn_s_setprio(0);
            }
        }
        if (careful || p0 >= p1) break;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < DS; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) top = largest_of(top, acc[i][j]);
        const bool lost = __any(R.live && top != top);
        wild = __any(!(top < __builtin_inff()));
        if (l == 0) M.range[0][w] = lost;
        __syncthreads();
        if (!__builtin_amdgcn_readfirstlane(M.range[0][0] | M.range[0][1] | M.range[0][2] | M.range[0][3])) break;
        idp = INT32_MIN / 2;
        blk = block_of(p0, bad);
        fetch(lds, A.kv.k, ko, p0, blk);
        fetch(lds + TB, A.kv.v, vo, p0, blk);
    }
    if (odd0 < odd1) {
        wild = true;
        idp = INT32_MIN / 2;
        for (int p = odd0; p < odd1; p += BN) {
            blk = block_of(p, bad);
            __syncthreads();   // every wave is done with the buffer and the flags
            fetch(lds, A.kv.v, vo, p, blk);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            look(lds, p, 0);
            __syncthreads();
            if ((found(0) & 2) && p < whi && p + BN > wlo) add_odd(lds, p, bad);
        }
    }
    sum = add_halves(sum);
    if (!R.live) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (nsplit == 1 && !A.parts_sh) {
        uint16_t *o = (uint16_t *)a.out + (int64_t)R.tok * a.out_token + R.head * a.out_head + 4 * hh;
#pragma unroll
        for (int i = 0; i < DS; i++)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                uint2 v = make_uint2(pack2<T>(acc[i][j] * inv, acc[i][j + 1] * inv), pack2<T>(acc[i][j + 2] * inv, acc[i][j + 3] * inv));
                if (sum == 0.0f) v = make_uint2(0, 0);
                *(uint2 *)(o + 32 * i + 2 * j) = v;
            }
        if (a.lse && hh == 0) a.lse[(int64_t)R.tok * a.heads + R.head] = sum == 0.0f ? -__builtin_inff() : (mb + __builtin_amdgcn_logf(sum)) * ATT_LN2;
        return;
    }
    const int64_t row = (shared ? 0 : A.at_tile) + ((int64_t)split * a.ntok + R.tok) * a.heads + R.head;
    if (hh == 0) A.pm[row] = make_float2(mb, wild ? -sum : sum);
    if (sum == 0.0f) return;
    float *o = A.po + row * D + 4 * hh;
#pragma unroll
    for (int i = 0; i < DS; i++)
#pragma unroll
        for (int j = 0; j < 16; j += 4) *(f4 *)(o + 32 * i + 2 * j) = f4{acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3]};
}

// Few rows (up to 16 per key/value head: single tokens, a few drafted ones): the cache's bytes are the bound, so a workgroup takes a chunk
// of positions, its waves runs of 32 in turn, keys and values straight into registers; a run's keys give their
// registers to the next run's as soon as its scores are there, its values after the second product. S^T = K Q^T and O^T = V^T P^T as in k_attn_tile, on 16 x 16 x 32
// products, the weights rounded to the cache's type there too; V^T is put together from rows by byte permutes (32 per run of 32 positions, hidden
// behind the loads). The waves join through LDS, the chunks in k_attn_join. Measured: one token over 100000 positions of 4 key/value heads
// of 128, 204.8 MB in 41 us, 5.0 TB/s (a copy of 1 GB reaches 5.06); 7 tokens over 2048 shared positions 7.9 us, latency. Two waves per SIMD:
// a third leaves too few registers for the loads under way (52 us instead of 43).
template <int T> __device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
    if (T == MMOE_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ float max_quarters(float x) { x = fmaxf(x, __shfl_xor(x, 16, 64)); return fmaxf(x, __shfl_xor(x, 32, 64)); }
__device__ __forceinline__ float add_quarters(float x) { x += __shfl_xor(x, 16, 64); return x + __shfl_xor(x, 32, 64); }

template <int D> struct AttFewMem {
    union {
        __attribute__((aligned(16))) float joint[4][16][D + 4];
        int starts[MMOE_KV_MAXSEQ + 1];
    };
    float2 stat[4][16];
};
template <int T, int D, bool CAP, bool BIAS>
__device__ __forceinline__ void att_few(const AttArgs &A, const bool shared, const unsigned block, AttFewMem<D> &M) {
    constexpr int KS = D / 32, E = D / 16;   // products over the dims, values of a row per lane
    const mmoe_attn_args &a = A.a;
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = l & 15, g = l >> 4;
    const unsigned rest = A.by_kv(block), v = (shared ? A.by_split_sh : A.by_chunks)(rest);
    const int kvh = block - rest * A.kv.heads, c = rest - v * (shared ? A.split_sh : A.chunks);
    AttTileAt at;
    int from, end;
    bool whole = false;   // the rows' only result
    if (shared) {
        at.s = 0; at.t0 = 0; at.row0 = (int)v * 16; at.rows = att_start(a, a.nseq) * A.group;
        from = c * A.chunk; end = min(from + A.chunk, a.shared);
    } else {
        at.s = (int)v; at.t0 = att_start(a, at.s); at.row0 = 0;
        int tokens = att_start(a, at.s + 1) - at.t0;
        at.rows = min(tokens, a.max_q) * A.group;
        if (at.rows > A.few || tokens < 1) return;
        AttChunks ch = att_chunks(A, at.s, tokens);
        if (c >= ch.n) return;
        whole = ch.n == 1 && !A.parts_sh;
        from = ch.from + c * A.chunk; end = min(from + A.chunk, ch.to);
    }
    if (at.row0 >= at.rows) return;
    const int32_t *table = a.table + (int64_t)at.s * a.width;
    auto ids = [&](int p) { return table[min((p + 16 * (l & 1)) >> A.sh, a.width - 1)]; };   // lane i % 2: positions p + 16 i ..
    // keys: lane (g, n) row n, dims 32 s + 8 g ..; values: rows 4 g + i, dims E n ..
    const uint32_t ko = (uint32_t)(n * A.kv.token_stride + 8 * g) * 2;
    uint32_t vo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) vo[i] = (uint32_t)((4 * g + i) * A.kv.token_stride + E * n) * 2;
    struct Run { u4 k[2][KS]; uint32_t v[2][4][E / 2]; unsigned bad; } r;
    auto place = [&](const void *base, int p, int id, int u) {
        int blk = __builtin_amdgcn_readlane(id, u);
        if ((unsigned)blk >= (unsigned)A.kv.nblocks) blk = 0;
        return (gb *)base + (blk * A.kv.block_stride + kvh * A.kv.head_stride + ((p + 16 * u) & (A.kv.block_size - 1)) * A.kv.token_stride) * 2;
    };
    auto load_k = [&](int p, int id) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            gb *kp = place(A.kv.k, p, id, u);
#pragma unroll
            for (int s = 0; s < KS; s++) r.k[u][s] = *(const gu4 *)(kp + ko + 64 * s);
        }
    };
    auto load_v = [&](int p, int id) {
        r.bad = (unsigned)__ballot((unsigned)id >= (unsigned)A.kv.nblocks) & 3u;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            gb *vp = place(A.kv.v, p, id, u);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (E == 8) {
                    u4 v = *(const gu4 *)(vp + vo[i]);
#pragma unroll
                    for (int x = 0; x < E / 2; x++) r.v[u][i][x] = v[x & 3];
                } else {
                    typedef uint32_t u2v __attribute__((ext_vector_type(2)));
                    u2v v = *(const __attribute__((address_space(1))) u2v *)(vp + vo[i]);
                    r.v[u][i][0] = v[0]; r.v[u][i][1] = v[1];
                }
            }
        }
    };
    AttRow R = att_row(A, at, at.row0 + n, kvh);
    // Unless rows begin at limits of their own, `from` is where they begin: the first run comes while they look for their limits
    // (one token over 100000 positions 46.8 us instead of 47.7 for the call, 64 over up to 3000 46.8 instead of 48.1)
    const bool early = !a.lo && a.window <= 0;
    int p = from + 32 * w, id = 0, next = 0;
    if (early) { id = ids(p); next = ids(p + 128); }
    const AttSeq sq = att_seq(A, shared, at, M.starts, R);
    if (early && p < end) { load_k(p, id); load_v(p, id); }
    att_limits(A, shared, sq, R);
    u4 q[KS];
    {
        const uint16_t *qp = (const uint16_t *)a.q + (int64_t)R.tok * a.q_token + R.head * a.q_head + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = *(const gu4 *)(qp + 32 * s);
    }
    const float slope = BIAS ? a.slopes[R.head] * ATT_LOG2E : 0.0f;
    const bool some = R.live && R.lo < R.hi;
    const int seen = wave_min(some ? R.lo : INT32_MAX);   // the first position that any row sees
    int p0 = max(from, seen & ~31), p1 = min(end, wave_max(some ? R.hi : 0));
    if (p0 >= p1) p0 = p1 = 0;   // nothing seen (p0 may be close to the largest int: no wave's first run is counted from it)
    const int inlo = wave_max(R.live ? R.lo : 0), inhi = wave_min(R.live ? R.hi : INT32_MAX);
    f4 acc[E];
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = f4{0, 0, 0, 0};
    float m = -__builtin_inff(), mb = 0.0f, sum = 0.0f;
    int odd0 = INT32_MAX, odd1 = 0;         // the runs in which some row may see a value that was zeroed (as in att_tile)
    bool careful = false, wild = false;     // every run's values are looked at; results may not be finite

    auto look = [&](int p) {   // the run's values: 1 if some are not finite, 2 if a row may see one
        uint32_t o = 0, see = 0;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t mine = 0;
#pragma unroll
                for (int x = 0; x < E / 2; x++) mine |= odd_pair<T>(r.v[u][i][x]);
                const int at = p + 16 * u + 4 * g + i;
                o |= mine;
                see |= at >= seen && at < p1 ? mine : 0;
            }
        return (__any((o & 0x80008000u) != 0) ? 1 : 0) | (__any((see & 0x80008000u) != 0) ? 2 : 0);
    };
    auto step = [&](int p, auto &&after_scores) {
        f4 s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            s[u] = f4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; k++) s[u] = mfma16<T>(r.k[u][k], q[k], s[u]);
        }
        after_scores();
        const float dist = BIAS ? (float)(R.pos - p - 4 * g) : 0.0f;
        const bool part = p < inlo || p + 32 > inhi || r.bad;
        float mt = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float x = s[u][j] * A.s1;
                if (CAP) x = fmaf(-2.0f * A.s2, __builtin_amdgcn_rcpf(1.0f + exp2_(x)), A.s2);
                if (BIAS) x = fmaf(-slope, fabsf(dist - (float)(16 * u + j)), x);
                int at = p + 16 * u + 4 * g + j;
                if (part) x = at >= R.lo && at < R.hi && !((r.bad >> u) & 1) ? x : -__builtin_inff();
                s[u][j] = x;
                mt = fmaxf(mt, x);
            }
        mt = max_quarters(mt);
        if (__any(mt - m > 8.0f)) {
            const float mn = fmaxf(m, mt), bn = lowered<T>(mn == -__builtin_inff() ? 0.0f : mn), al = m == -__builtin_inff() ? 0.0f : exp2_(mb - bn);
            m = mn; mb = bn; sum *= al;
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] *= al;
        }
        u4 pf;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                float e0 = exp2_(s[u][j] - mb), e1 = exp2_(s[u][j + 1] - mb);
                sum += e0 + e1;
                pf[2 * u + (j >> 1)] = pack2<T>(e0, e1);
            }
        const int odd = careful || part ? look(p) : 0;
        if (odd) {
            if (odd & 2) { odd0 = min(odd0, p); odd1 = p + 1; }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int x = 0; x < E / 2; x++) r.v[u][i][x] = only_finite<T>(r.v[u][i][x]);
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            u4 f;
#pragma unroll
            for (int x = 0; x < 4; x++)   // positions 2 x and 2 x + 1 of the lane's eight
                f[x] = __builtin_amdgcn_perm(r.v[x >> 1][2 * (x & 1) + 1][e >> 1], r.v[x >> 1][2 * (x & 1)][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
            acc[e] = mfma16<T>(f, pf, acc[e]);
        }
    };
    if (!early) {
        p = p0 + 32 * w;
        id = ids(p); next = ids(p + 128);
        if (p < p1) { load_k(p, id); load_v(p, id); }
    }
    const int start = p;
    while (p < p1) {
        for (; p + 128 < p1; p += 128) {
            step(p, [&] { load_k(p + 128, next); });
            load_v(p + 128, next);
            next = ids(p + 256);
        }
        step(p, [] {});
        if (careful) break;
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 4; j++) top = largest_of(top, acc[e][j]);
        wild = __any(!(top < __builtin_inff()));
        if (!__any(R.live && top != top)) break;
        careful = true;   // once more
        m = -__builtin_inff(); mb = sum = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = f4{0, 0, 0, 0};
        p = start;
        id = ids(p); next = ids(p + 128);
        load_k(p, id); load_v(p, id);
    }
    if (odd0 < odd1) {   // through the wave's part of LDS
        wild = true;
        uint32_t *t = (uint32_t *)M.joint[w];
        for (p = odd0; p < odd1; p += 128) {
            load_v(p, ids(p));
            if (!(look(p) & 2)) continue;
            asm volatile("" ::: "memory");   // (words and floats in the same place)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int x = 0; x < E / 2; x++) t[(16 * u + 4 * g + i) * (D / 2) + n * (E / 2) + x] = r.v[u][i][x];
            __builtin_amdgcn_wave_barrier();   // a wave's LDS operations stay in order
#pragma unroll 1
            for (int k = 0; k < 32; k++) {
                const bool see = p + k >= R.lo && p + k < R.hi && !((r.bad >> (k >> 4)) & 1);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        uint32_t v = t[k * (D / 2) + ((4 * g + j) * E + e) / 2] >> (16 * (e & 1));
                        acc[e][j] += see && odd16<T>(v) ? half_to_f<T>(v & 0xffff) : 0.0f;
                    }
            }
        }
        asm volatile("" ::: "memory");
    }
    sum = add_quarters(sum);
    if (g == 0) M.stat[w][n] = make_float2(mb, wild ? -sum : sum);   // a negative sum: look at the results also where their weight is 0
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < E; e += 4) *(f4 *)&M.joint[w][n][(4 * g + j) * E + e] = f4{acc[e][j], acc[e + 1][j], acc[e + 2][j], acc[e + 3][j]};
    __syncthreads();
    // rows of 16 threads, D / 16 dims each
    const int jr = threadIdx.x >> 4, d = (threadIdx.x & 15) * E, row = at.row0 + jr;
    if (row >= at.rows) return;
    float2 st[4];
    float mx = -__builtin_inff(), total = 0.0f, o[E] = {};
    bool any = false;   // of them not finite, perhaps
#pragma unroll
    for (int i = 0; i < 4; i++) {
        st[i] = M.stat[i][jr];
        if (st[i].y != 0.0f) mx = fmaxf(mx, st[i].x);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (st[i].y == 0.0f) continue;
        float e = exp2_(st[i].x - mx);
        total = fmaf(fabsf(st[i].y), e, total);
        any |= st[i].y < 0.0f;
#pragma unroll
        for (int x = 0; x < E; x++) o[x] = fmaf(e, M.joint[i][jr][d + x], o[x]);
    }
    if (any)   // results that are not finite count whatever their weight
#pragma unroll 1
        for (int x = 0; x < E; x++) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e = st[i].y != 0.0f ? exp2_(st[i].x - mx) : 0.0f, y = M.joint[i][jr][d + x];
                if (e != 0.0f) sum = fmaf(e, y, sum); else if (st[i].y != 0.0f) sum += only_odd(y);
            }
#pragma unroll
            for (int y = 0; y < E; y++) if (y == x) o[y] = sum;
        }
    const int j = (int)A.by_group(row), tok = at.t0 + j, head = kvh * A.group + row - j * A.group;
    if (shared) {   // tokens past max_q have no partial results
        int s = max(count_le(a.qstart, a.nseq, tok) - 1, 0);
        if (tok - a.qstart[s] >= a.max_q) return;
    }
    if (whole) {
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        uint32_t *op = (uint32_t *)((uint16_t *)a.out + (int64_t)tok * a.out_token + head * a.out_head + d);
#pragma unroll
        for (int x = 0; x < E; x += 2) op[x / 2] = total == 0.0f ? 0u : pack2<T>(o[x] * inv, o[x + 1] * inv);
        if (a.lse && d == 0) a.lse[(int64_t)tok * a.heads + head] = total == 0.0f ? -__builtin_inff() : (mx + __builtin_amdgcn_logf(total)) * ATT_LN2;
        return;
    }
    const int64_t at_row = shared ? ((int64_t)c * a.ntok + tok) * a.heads + head : A.at_few + ((int64_t)c * a.nseq + at.s) * 16 * A.kv.heads + j * a.heads + head;
    if (d == 0) A.pm[at_row] = make_float2(mx, any ? -total : total);
    if (total == 0.0f) return;
#pragma unroll
    for (int x = 0; x < E; x += 4) *(f4 *)(A.po + at_row * D + d + x) = f4{o[x], o[x + 1], o[x + 2], o[x + 3]};
}

// One launch for everything, the long work first. With no row tiles of 128 in it a kernel of its own: fewer registers, more waves.
template <int T, int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256, 2) k_attn_few(AttArgs A) {
    __shared__ AttFewMem<D> M;
    const unsigned b = blockIdx.x;
    const bool shared = b < A.n_sh;
    att_few<T, D, CAP, BIAS>(A, shared, shared ? b : b - A.n_sh, M);
}
template <int T, int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256, 2) k_attn_tile(AttArgs A) {
    __shared__ union { AttTileMem<D> tile; AttFewMem<D> few; } M;
    const unsigned b = blockIdx.x;
    const bool shared = b < A.n_sh;
    if (shared ? !A.sh_few : b < A.n_sh + A.n_tile) att_tile<T, D, CAP, BIAS>(A, shared, shared ? b : b - A.n_sh, M.tile);
    else att_few<T, D, CAP, BIAS>(A, shared, shared ? b : b - A.n_sh - A.n_tile, M.few);
}

// The partial results of a row: their maxima and sums give each a weight. D / 4 lanes read a part; with all, every such group of the
// workgroup works on one row (the loads of a row's parts are what there is to wait for), else each has its own (up to ATT_PER parts).
// few_only: the rows are those of the sequences of few rows, 16 per key/value head.
// 1024 rows of 18 parts 7.8 us, 16 rows of 98 parts 5.9, 28 of 9 3.8: latency of two dependent loads (a part's maximum and sum, its values).
#define ATT_PARTS 1024     // most partial results of a row
#define ATT_PER 16
template <int T, int D>
__global__ void __launch_bounds__(1024) k_attn_join(AttArgs A, int all, int few_only) {
    constexpr int LPR = D / 4;
    const mmoe_attn_args &a = A.a;
    __shared__ float red[2][16], wt[ATT_PARTS];
    __shared__ int odd[16];
    __shared__ union { __attribute__((aligned(16))) float acc[1024 / LPR][D]; int starts[MMOE_KV_MAXSEQ + 1]; } M;
    const int gr = blockDim.x / LPR, gi = threadIdx.x / LPR, x = (threadIdx.x % LPR) * 4, row0 = all ? blockIdx.x : blockIdx.x * gr + gi;
    int tok, head, s, t0, tokens;
    bool on = true;
    if (few_only) {
        const int per = 16 * A.kv.heads;
        s = row0 / per;
        on = s < a.nseq;
        if (!on) s = 0;
        t0 = att_start(a, s); tokens = att_start(a, s + 1) - t0;
        const int r = row0 - s * per, j = (int)A.by_heads(r);
        on = on && min(tokens, a.max_q) * A.group <= A.few && j < tokens;
        tok = t0 + j; head = r - j * a.heads;
    } else {
        tok = (int)A.by_heads(row0); head = row0 - tok * a.heads;
        if (all) s = max(count_wave(a.nseq, [&](int i) { return a.qstart[i] <= tok; }) - 1, 0);
        else {
            for (int i = threadIdx.x; i <= a.nseq; i += blockDim.x) M.starts[i] = a.qstart[i];
            __syncthreads();
            s = max(count_le(M.starts, a.nseq, tok) - 1, 0);
        }
        on = tok < att_start(a, a.nseq);
        t0 = att_start(a, s); tokens = att_start(a, s + 1) - t0;
    }
    if (!on || tok < t0 || tok - t0 >= min(tokens, a.max_q)) return;   // (with all: the whole workgroup)
    const bool few = min(tokens, a.max_q) * A.group <= A.few;
    const int parts = A.parts_sh + (few ? att_chunks(A, s, tokens).n : A.split);
    if (parts == 1) return;   // written by the one that had it
    const int64_t rows = (int64_t)a.ntok * a.heads, row = (int64_t)tok * a.heads + head;
    const int64_t own = few ? A.at_few + (int64_t)s * 16 * A.kv.heads + (tok - t0) * a.heads + head : A.at_tile + row;
    const int64_t by = few ? (int64_t)a.nseq * 16 * A.kv.heads : rows;
    auto part = [&](int p) { return p < A.parts_sh ? p * rows + row : own + (p - A.parts_sh) * by; };
    float m = -__builtin_inff(), sum = 0.0f;
    f4 o = {0, 0, 0, 0};
    bool some = false;
    if (all) {
        const int l = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
        float2 v[ATT_PARTS / 256];
#pragma unroll
        for (int i = 0; i < ATT_PARTS / 256; i++) {
            int p = threadIdx.x + i * blockDim.x;
            v[i] = p < parts ? A.pm[part(p)] : make_float2(0, 0);
            if (v[i].y != 0.0f) m = fmaxf(m, v[i].x);
        }
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        if (l == 0) red[0][w] = m;
        __syncthreads();
        for (int i = 0; i < nw; i++) m = fmaxf(m, red[0][i]);
#pragma unroll
        for (int i = 0; i < ATT_PARTS / 256; i++) {
            int p = threadIdx.x + i * blockDim.x;
            float e = v[i].y != 0.0f ? exp2_(v[i].x - m) : 0.0f;
            const bool look = v[i].y < 0.0f && e == 0.0f;   // results that are not finite count whatever their weight
            if (p < parts) wt[p] = look ? -1.0f : e;
            some |= look;
            sum = fmaf(fabsf(v[i].y), e, sum);
        }
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
        some = __any(some);
        if (l == 0) { red[1][w] = sum; odd[w] = some; }
        __syncthreads();
        sum = 0.0f;
        for (int i = 0; i < nw; i++) { sum += red[1][i]; some |= odd[i] != 0; }
#pragma unroll 8
        for (int p = gi; p < parts; p += gr) {
            float e = wt[p];
            f4 y = e <= 0.0f ? f4{0, 0, 0, 0} : *(const f4 *)(A.po + part(p) * D + x);
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = fmaf(e, y[i], o[i]);
        }
        if (some)
            for (int p = gi; p < parts; p += gr) {
                if (wt[p] != -1.0f) continue;
                f4 y = *(const f4 *)(A.po + part(p) * D + x);
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] += only_odd(y[i]);
            }
        *(f4 *)&M.acc[gi][x] = o;
        __syncthreads();
        if (gi) return;
        for (int i = 1; i < gr; i++) o += *(const f4 *)&M.acc[i][x];
    } else {
        float2 v[ATT_PER];   // every part's, all loads under way at once
#pragma unroll
        for (int p = 0; p < ATT_PER; p++) v[p] = p < parts ? A.pm[part(p)] : make_float2(0, 0);
#pragma unroll
        for (int p = 0; p < ATT_PER; p++) if (v[p].y != 0.0f) m = fmaxf(m, v[p].x);
#pragma unroll
        for (int p = 0; p < ATT_PER; p++) {
            f4 y = v[p].y != 0.0f ? *(const f4 *)(A.po + part(p) * D + x) : f4{0, 0, 0, 0};
            float e = v[p].y != 0.0f ? exp2_(v[p].x - m) : 0.0f;
            sum = fmaf(fabsf(v[p].y), e, sum);
            some |= v[p].y < 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = fmaf(e, y[i], o[i]);
        }
        if (some) {   // results that are not finite count whatever their weight
            o = f4{0, 0, 0, 0};
#pragma unroll 1
            for (int p = 0; p < parts; p++) {
                const float2 v = A.pm[part(p)];
                if (v.y == 0.0f) continue;
                const float e = exp2_(v.x - m);
                const f4 y = *(const f4 *)(A.po + part(p) * D + x);
#pragma unroll
                for (int i = 0; i < 4; i++) if (e != 0.0f) o[i] = fmaf(e, y[i], o[i]); else o[i] += only_odd(y[i]);
            }
        }
    }
    const float inv = 1.0f / sum;
    uint2 v = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
    if (sum == 0.0f) v = make_uint2(0, 0);
    *(uint2 *)((uint16_t *)a.out + (int64_t)tok * a.out_token + head * a.out_head + x) = v;
    if (a.lse && x == 0) a.lse[row] = sum == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(sum)) * ATT_LN2;
}
