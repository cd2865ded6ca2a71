// drafts.h -- kernels for drafted tokens (what each follows, which are accepted) and for blocks that sequences share, copy and give back
// (drafts.hip).
#pragma once
#include "paged.h"

// Where sequence s's new tokens begin and how many of them lie inside the arrays, whatever qstart holds; what was cached before all of them
struct NewTokens { int t0, n, ctx; };
__device__ __forceinline__ NewTokens new_tokens(const int32_t *qstart, const int32_t *len, int s, int ntok) {
    const int t0 = min(max(qstart[s], 0), ntok), t1 = max(qstart[s + 1], t0);
    return {t0, min(t1, ntok) - t0, len[s] - (t1 - t0)};
}

// ------------------------------------------------------------------------------------------------------
// What drafted tokens follow (mmoe_tree_plan)
// ------------------------------------------------------------------------------------------------------
// A workgroup per sequence, a wave per word of 64 nodes, a lane per node. Within a word by steps that double (what a node's 2^i-th ancestor
// follows, it follows), through the lanes: six steps at most, which leave each node the ancestors of its own word and the node of an earlier word
// that the last of them follows, if any. From there every node goes from word to word by itself, through LDS (word by word for all nodes at once, with a
// barrier for each: 7.3 us instead of 4.9 below). A wave's rows of bits lie one behind the other and are written so. Bound by latency: the launch,
// the tree's place, its parents, the steps. Measured: 64 trees of 10 to 40 nodes 4.1 us, 200 of 300 to 512 nodes 4.9 us (5.9 MB, 1.2 TB/s).
template <int W>
__global__ void __launch_bounds__(64 * W) k_tree_plan(mmoe_tree_plan_args a) {
    __shared__ uint64_t words[W * 64];       // each node's bits of its own word
    __shared__ int outs[W * 64];             // and the node of an earlier word
    __shared__ uint64_t rows[W][W * 64];     // a wave's rows as they are written
    const int s = blockIdx.x, i = threadIdx.x, l = i & 63, wave = __builtin_amdgcn_readfirstlane(i >> 6);
    const NewTokens q = a.nseq ? new_tokens(a.qstart, a.len, s, a.ntok) : NewTokens{0, 0, 0};
    const int n = min(q.n, 64 * a.words);
    int out = -1;
    if (i < n) out = a.parent[q.t0 + i];
    if (out < 0 || out >= i) out = -1;   // (before the subtraction, which would make a lane of a number near the smallest: a node may then follow itself)
    int to = out - 64 * wave;            // in the word: its lane, below the node's own, so that the steps end
    uint64_t own = 1ull << l;
    while (__any(to >= 0)) {
        const int from = max(to, 0);
        const uint64_t more = (uint64_t)(uint32_t)__shfl((int)(own >> 32), from, 64) << 32 | (uint32_t)__shfl((int)own, from, 64);
        const int next = __shfl(to, from, 64), past = __shfl(out, from, 64);
        if (to >= 0) { own |= more; to = next; out = past; }
    }
    uint64_t b[W] = {};
    if (W > 1) {
        words[i] = own; outs[i] = out;
        __syncthreads();
    }
    int depth = __popcll(own) - 1;
#pragma unroll
    for (int w = W - 1; w >= 0; w--) {
        if (w == wave) b[w] = own;
        if (w < wave && out >= 64 * w) {
            b[w] = words[out]; out = outs[out];
            depth += __popcll(b[w]);
        }
    }
    if (i < n) a.pos[q.t0 + i] = q.ctx + depth;
    // row by row, `words` words each; the places of a row turned by its number, so that the lanes' places lie in different banks
    const int per = a.words, live = min(max(n - 64 * wave, 0), 64) * per;
#pragma unroll
    for (int w = 0; w < W; w++) rows[wave][l * W + ((w + l) & (W - 1))] = b[w];
    __builtin_amdgcn_wave_barrier();
    const unsigned by = (65536 + per - 1) / per;   // x / per for x < 512
    uint64_t *bits = a.bits + (int64_t)(q.t0 + 64 * wave) * per;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int x = 64 * w + l, r = (int)(x * by >> 16), c = x - r * per;
        if (x < live) bits[x] = rows[wave][r * W + ((c + r) & (W - 1))];
    }
    // nodes past the words, and tokens of no sequence
    for (int t = q.t0 + n + i; t < q.t0 + q.n; t += 64 * W) {
        a.pos[t] = 0;
        for (int w = 0; w < a.words; w++) a.bits[(int64_t)t * a.words + w] = 0;
    }
    for (int64_t t = min(max(a.qstart[a.nseq], 0), a.ntok) + (int64_t)s * 64 * W + i; t < a.ntok; t += (int64_t)gridDim.x * 64 * W) {
        a.pos[t] = 0;
        for (int w = 0; w < a.words; w++) a.bits[t * a.words + w] = 0;
    }
}

// ------------------------------------------------------------------------------------------------------
// Which drafted tokens stay (mmoe_tree_accept)
// ------------------------------------------------------------------------------------------------------
// A workgroup per sequence: every node that is what the model chose behind its parent offers itself to it, the lowest one wins (so the order of the
// atomics does not matter); then the walk from node 0 is a chain of reads from LDS. Latency: 2.4 to 3.0 us for 5 and for 64 sequences.
__global__ void __launch_bounds__(128) k_tree_accept(mmoe_tree_accept_args a) {
    __shared__ int child[MMOE_TREE_MAX];
    const int s = blockIdx.x;
    const NewTokens q = new_tokens(a.qstart, a.len, s, a.ntok);
    const int n = min(q.n, MMOE_TREE_MAX);
    for (int i = threadIdx.x; i < n; i += 128) child[i] = INT32_MAX;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 128) {
        const int p = a.parent[q.t0 + i];
        if (p >= 0 && p < i && a.token[q.t0 + i] == a.next[q.t0 + p]) atomicMin(&child[p], i);
    }
    __syncthreads();
    if (threadIdx.x) return;
    int count = 0, last = 0;
    for (int i = 0; i < n; i = child[i]) {   // (a child lies behind its parent: the walk ends)
        a.kept[q.t0 + count++] = q.ctx + i;
        last = i;
    }
    a.count[s] = count;
    a.last[s] = n ? a.next[q.t0 + last] : -1;
    a.ctx[s] = q.ctx + count;
}

// ------------------------------------------------------------------------------------------------------
// Blocks in every layer (mmoe_kv_compact, mmoe_kv_copy)
// ------------------------------------------------------------------------------------------------------
// A position is heads * pieces pieces of 16 bytes, numbered head by head. The layers' arrays differ in their pointers only.
struct PageArgs {
    mmoe_kv_cache kv;                  // the layers' strides and sizes (k and v unused)
    int sh, esize, pieces, all;        // log2 of the block size, bytes of a value, pieces of a head, of a position
    Div by_pieces;
    void *base[2 * MMOE_KV_MAXLAYERS]; // keys and values of each layer
};
__device__ __forceinline__ int64_t page_at(const PageArgs &P, int block, int at, int piece) {   // in bytes
    const int head = (int)P.by_pieces(piece);
    return (block * P.kv.block_stride + head * P.kv.head_stride + at * P.kv.token_stride) * P.esize + (int64_t)(piece - head * P.pieces) * 16;
}

// Kept positions moved together. Entry j goes from k[j] to k[0] + j <= k[j], so that writing it touches the source of no later one: a
// workgroup goes through the list in steps of as many entries as its threads hold, all of a step read before any is written; positions and blocks of the
// next step are looked up while this one's values are on their way. A workgroup has `lanes` pieces of every position (of one array), so the
// arrays and the pieces are what runs side by side. Bound by memory where lists are long: one sequence of 20000 positions cut to 8000 in 24 layers, 4
// heads of 128, 786 MB: 171 us, 4.6 TB/s (a copy reaches 5.1); without the look-ups a step ahead 420; with the values a step ahead too, no faster. What
// a draft leaves behind (64 sequences, a few tokens each, 12.6 MB): 5.7 us, five loads that depend on one another.
#define KC_U 8
template <int TH>
__global__ void __launch_bounds__(TH) k_kv_compact(mmoe_kv_compact_args a, PageArgs P, int lanes, int units, Div by_lanes, Div by_units, Div by_arrays, int arrays) {
    // the arrays first: a position's pieces then lie on one die wherever the number of arrays is a multiple of the dies'
    const unsigned rest = by_arrays(blockIdx.x), s = by_units(rest);
    const int array = blockIdx.x - rest * arrays, unit = rest - s * units;
    const int first = a.first[s], n = a.count[s];
    if (first < 0 || first >= a.nkept || n < 2) return;
    const int count = min(n, a.nkept - first), per = (int)by_lanes(TH), e = (int)by_lanes(threadIdx.x);
    const int piece = unit * lanes + threadIdx.x - e * lanes, bs1 = P.kv.block_size - 1;
    const bool on = e < per && piece < P.all;
    const int32_t *k = a.kept + first, *table = a.table + (int64_t)s * a.width;
    const int to0 = k[0];
    uint8_t *base = (uint8_t *)P.base[array];
    auto block = [&](int64_t p) { return p < 0 || (p >> P.sh) >= a.width ? -1 : table[p >> P.sh]; };
    struct Step { int from[KC_U], b0[KC_U], b1[KC_U]; };
    auto positions = [&](Step &x, int j0) {
#pragma unroll
        for (int u = 0; u < KC_U; u++) {
            const int j = j0 + u * per + e;
            x.from[u] = on && j < count ? k[j] : -1;
        }
    };
    auto blocks = [&](Step &x, int j0) {
#pragma unroll
        for (int u = 0; u < KC_U; u++) {
            const int64_t t = (int64_t)to0 + j0 + u * per + e;
            const bool moves = x.from[u] > t;
            x.b0[u] = moves ? block(x.from[u]) : -1;
            x.b1[u] = moves ? block(t) : -1;
        }
    };
    Step now, then;
    positions(now, 1);
    blocks(now, 1);
    for (int j0 = 1; j0 < count; j0 += per * KC_U) {
        const int j1 = j0 + per * KC_U;
        u4 x[KC_U];
#pragma unroll
        for (int u = 0; u < KC_U; u++) {
            if ((unsigned)now.b0[u] >= (unsigned)P.kv.nblocks || (unsigned)now.b1[u] >= (unsigned)P.kv.nblocks) { now.b1[u] = -1; continue; }
            x[u] = *(const gu4 *)(base + page_at(P, now.b0[u], now.from[u] & bs1, piece));
        }
        if (j1 < count) { positions(then, j1); blocks(then, j1); }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every wave's values are there before any is written over
        __syncthreads();
#pragma unroll
        for (int u = 0; u < KC_U; u++) if (now.b1[u] >= 0) *(gu4 *)(base + page_at(P, now.b1[u], (to0 + j0 + u * per + e) & bs1, piece)) = x[u];
        now = then;
    }
}

// A workgroup has KY_U KY_T pieces of 16 bytes of one block of one array, all on their way at once. Bound by memory: 48 begun blocks of a beam
// search's step in 24 layers, 89 MB: 16 us, 5.5 TB/s with what the caches hold; 32 of 16 positions: 4.5 us, latency.
#define KY_T 256
#define KY_U 8
__global__ void __launch_bounds__(KY_T) k_kv_copy(mmoe_kv_copy_args a, PageArgs P, int units, Div by_units, Div by_arrays, int arrays) {
    const unsigned rest = by_units(blockIdx.x), i = by_arrays(rest);
    const int unit = blockIdx.x - rest * units, array = rest - i * arrays;
    const int from = a.copy_from[i], to = a.copy_to[i], bs = P.kv.block_size;
    const int count = a.copy_count ? min(max(a.copy_count[i], 0), bs) : bs;
    if ((unsigned)from >= (unsigned)P.kv.nblocks || (unsigned)to >= (unsigned)P.kv.nblocks || from == to) return;
    uint8_t *base = (uint8_t *)P.base[array];
    u4 x[KY_U];
    int64_t at[KY_U];
#pragma unroll
    for (int u = 0; u < KY_U; u++) {   // head by head, positions within, pieces within those
        const int item = (unit * KY_U + u) * KY_T + threadIdx.x, row = (int)P.by_pieces(item), head = row >> P.sh, pos = row & (bs - 1);
        at[u] = -1;
        if (head >= P.kv.heads || pos >= count) continue;
        at[u] = (head * P.kv.head_stride + pos * P.kv.token_stride) * P.esize + (int64_t)(item - row * P.pieces) * 16;
        x[u] = *(const gu4 *)(base + from * P.kv.block_stride * P.esize + at[u]);
    }
#pragma unroll
    for (int u = 0; u < KY_U; u++) if (at[u] >= 0) *(gu4 *)(base + to * P.kv.block_stride * P.esize + at[u]) = x[u];
}

// ------------------------------------------------------------------------------------------------------
// Copies of sequences (mmoe_kv_fork)
// ------------------------------------------------------------------------------------------------------
// One workgroup settles which forks are made and which blocks they take (a prefix sum over them); the rows, which are independent, follow in the
// same launch or, where they have more than KO_ONE entries, in one of their own. Latency: the lengths, the list, the rows: 2.8 to 3.4 us for 64 beams and
// 32 samples (rows by waves 5.3, workgroups of 256 10).
// columns of a copy's row that are its source's
__device__ __forceinline__ int fork_cols(const mmoe_kv_fork_args &a, int sh, int n) { return n <= a.shared ? (n + a.block_size - 1) >> sh : n >> sh; }
__device__ __forceinline__ void fork_put(const mmoe_kv_fork_args &a, int sh, int dst, int c, int b) {
    a.table_out[(int64_t)dst * a.width + c] = b;
    if (c >= a.shared >> sh && (unsigned)b < (unsigned)a.nblocks) atomicAdd(&a.holders[b], 1);
}
#define KO_ONE 4096   // rows' entries that the one workgroup copies itself
template <int PER>
__global__ void __launch_bounds__(1024) k_kv_fork(mmoe_kv_fork_args a, int sh, int rows, Div by_width) {
    __shared__ int src_[PER * 1024], dst_[PER * 1024], len_[PER * 1024];
    __shared__ uint2 red[16];
    const int tid = threadIdx.x, i0 = tid * PER;
    const int nfree = min(max(a.nfree[0], 0), a.nblocks);
    int src[PER], dst[PER], n[PER], begun[PER];
    unsigned need[PER], sum = 0, zero = 0, total, z;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const bool in = i0 + i < a.nfork;
        src[i] = in ? a.src[i0 + i] : -1; dst[i] = in ? a.dst[i0 + i] : -1;
        const bool ok = (unsigned)src[i] < (unsigned)a.nseq && (unsigned)dst[i] < (unsigned)a.nseq;
        if (!ok) src[i] = -1;
        n[i] = ok ? a.ctx[src[i]] : 0;
        if (ok && a.at) n[i] = min(n[i], a.at[i0 + i]);
        n[i] = min(max(n[i], 0), a.width << sh);
        need[i] = (n[i] & (a.block_size - 1)) && n[i] > a.shared;
        begun[i] = need[i] ? a.table[(int64_t)src[i] * a.width + (n[i] >> sh)] : -1;
        sum += need[i];
    }
    scan2(sum, zero, &total, &z, red);   // (and every length has been read before one is written)
    if (tid == 0) a.nfree_out[0] = nfree - (int)min(total, (unsigned)nfree);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i0 + i >= a.nfork) continue;
        const unsigned at = sum;
        sum += need[i];
        const bool fits = sum <= (unsigned)nfree, takes = need[i] && fits;
        const int b = takes ? a.free_list[nfree - 1 - at] : -1;
        if (!fits) n[i] = 0;
        if (src[i] >= 0) {
            a.ctx_out[dst[i]] = n[i];
            if (takes) a.table_out[(int64_t)dst[i] * a.width + (n[i] >> sh)] = b;
        } else if ((unsigned)dst[i] < (unsigned)a.nseq) a.ctx_out[dst[i]] = 0;
        a.copy_from[i0 + i] = takes ? begun[i] : -1;
        a.copy_to[i0 + i] = b;
        a.copy_count[i0 + i] = takes ? n[i] & (a.block_size - 1) : 0;
        src_[i0 + i] = src[i]; dst_[i0 + i] = dst[i]; len_[i0 + i] = n[i];
    }
    if (!rows) return;
    __syncthreads();
    int b[KO_ONE / 1024], c[KO_ONE / 1024], to[KO_ONE / 1024];
#pragma unroll
    for (int u = 0; u < KO_ONE / 1024; u++) {   // every load under way at once
        const int item = u * 1024 + tid, i = (int)by_width(item);
        c[u] = item - i * a.width; to[u] = -1;
        if (i >= a.nfork || src_[i] < 0 || c[u] >= fork_cols(a, sh, len_[i])) continue;
        b[u] = a.table[(int64_t)src_[i] * a.width + c[u]];
        to[u] = dst_[i];
    }
#pragma unroll
    for (int u = 0; u < KO_ONE / 1024; u++) if (to[u] >= 0) fork_put(a, sh, to[u], c[u], b[u]);
}
__global__ void __launch_bounds__(256) k_kv_fork_rows(mmoe_kv_fork_args a, int sh) {
    const int src = a.src[blockIdx.x], dst = a.dst[blockIdx.x];
    if ((unsigned)src >= (unsigned)a.nseq || (unsigned)dst >= (unsigned)a.nseq) return;
    const int cols = fork_cols(a, sh, a.ctx_out[dst]);
    for (int c = threadIdx.x; c < cols; c += 256) fork_put(a, sh, dst, c, a.table[(int64_t)src * a.width + c]);
}

// ------------------------------------------------------------------------------------------------------
// Blocks given back (mmoe_kv_free)
// ------------------------------------------------------------------------------------------------------
// What sequences give up, one behind the other, is a list of places in the tables; a block goes back with the last of them that drops it to
// nobody. Three passes over that list with holders: every place drops a holder; of the places of a block that nobody holds now the last one marks
// it; the marked ones are appended in order. Sums and marks, not the order of the atomics, decide, so the list comes out the same every time. One
// workgroup, since the list is one; latency: 2.2 us for 5 sequences, 3.1 for 64 that give up a draft's blocks, 7.8 for 64 rows of a beam search that
// give up all of theirs (800 places, three rounds of atomics).
#define KF_U 4
template <int PER>
__global__ void __launch_bounds__(1024) k_kv_free(mmoe_kv_free_args a, int sh) {
    constexpr int NS = PER * 1024;
    __shared__ int first[NS + 1], col[NS];
    __shared__ uint2 red[16];
    const int tid = threadIdx.x, nt = blockDim.x, s0 = tid * PER, bs1 = a.block_size - 1, pre = a.shared >> sh, nfree = min(max(a.nfree[0], 0), a.nblocks);
    const int room = a.width << sh;
    unsigned old[PER], sum = 0, zero = 0, total, z;
    int len[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        old[i] = 0;
        if (s0 + i >= a.nseq) continue;
        const int ctx = min(max(a.ctx[s0 + i], 0), room);
        int k = min(ctx, max(a.keep[s0 + i], a.shared));
        if (a.holders && k < ctx && (k & bs1) && k > a.shared) {
            const int b = a.table[(int64_t)(s0 + i) * a.width + (k >> sh)];
            if ((unsigned)b < (unsigned)a.nblocks && a.holders[b] > 0) k = ctx;
        }
        len[i] = k;
        const int c0 = max((k + bs1) >> sh, pre), c1 = (ctx + bs1) >> sh;
        col[s0 + i] = c0;
        old[i] = (unsigned)max(c1 - c0, 0);
        sum = min(sum + old[i], (unsigned)KP_LIM);
    }
    scan2(sum, zero, &total, &z, red);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (s0 + i >= a.nseq) continue;
        a.len[s0 + i] = len[i];
        first[s0 + i] = (int)sum;
        sum = min(sum + old[i], (unsigned)KP_LIM);
    }
    __syncthreads();
    const int n = (int)total;
    auto id = [&](int j) {
        const int s = count_le(first, a.nseq, j) - 1;
        return a.table[(int64_t)s * a.width + col[s] + j - first[s]];
    };
    // KF_U places a thread, one behind the other; those of the first round stay in registers
    int b[KF_U];
    auto round = [&](int j0) {
#pragma unroll
        for (int u = 0; u < KF_U; u++) {
            const int j = j0 + tid * KF_U + u;
            b[u] = j < n ? id(j) : -1;
            if ((unsigned)b[u] >= (unsigned)a.nblocks) b[u] = -1;
        }
    };
    const bool once = n <= nt * KF_U;
    round(0);
    if (a.holders) {
        for (int j0 = 0; j0 < n; j0 += nt * KF_U) {
            if (j0) round(j0);
#pragma unroll
            for (int u = 0; u < KF_U; u++) if (b[u] >= 0) atomicSub(&a.holders[b[u]], 1);
        }
        __threadfence();
        __syncthreads();
        for (int j0 = 0; j0 < n; j0 += nt * KF_U) {
            if (!once) round(j0);
            int h[KF_U];
#pragma unroll
            for (int u = 0; u < KF_U; u++) h[u] = b[u] >= 0 ? __hip_atomic_load(&a.holders[b[u]], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
            for (int u = 0; u < KF_U; u++) if (h[u] < 0) atomicMin(&a.holders[b[u]], -2 - (j0 + tid * KF_U + u));
        }
        __threadfence();
        __syncthreads();
    }
    int at = nfree;
    for (int j0 = 0; j0 < n; j0 += nt * KF_U) {
        unsigned mine = 0, none = 0, all, z2;
        if (!once) round(j0);
#pragma unroll
        for (int u = 0; u < KF_U; u++) {
            const int j = j0 + tid * KF_U + u;
            if (b[u] < 0) continue;
            if (a.holders && __hip_atomic_load(&a.holders[b[u]], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != -2 - j) b[u] = -1;
            mine += b[u] >= 0;
        }
        scan2(mine, none, &all, &z2, red);
#pragma unroll
        for (int u = 0; u < KF_U; u++) {
            if (b[u] < 0) continue;
            if (at + (int)mine < a.nblocks) a.free_list[at + mine] = b[u];
            if (a.holders) a.holders[b[u]] = 0;
            mine++;
        }
        at = min(at + (int)all, a.nblocks);
    }
    if (tid == 0) a.nfree_out[0] = at;
}
