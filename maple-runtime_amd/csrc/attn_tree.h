// attn_tree.h -- attention of drafted tokens over the blocks (mmoe_attn_tree, drafts.hip).
//
// The row tiles are mmoe_attn_paged's (att_tile, with masks from the tokens' bits). What differs is who gets which: a draft makes few row tiles per
// sequence, each as long as the sequence, so that time goes by how evenly they are shared out. The row tiles' positions are cut into pieces of at most a
// number of steps (of TREE_BN positions) which is so chosen that there are no more pieces than the card has room for at once (two workgroups
// per compute unit): a few more would wait for a second round. Every workgroup finds its piece from the sequences' lengths themselves, so grid and
// workspace follow the numbers of workgroups and row tiles, not the bounds of the lengths.
#pragma once
#include <type_traits>
#include "paged.h"

// Partial results are kept in waves of 32 rows. Those over the shared positions come first, then sequence by sequence, of each what it has over its first
// positions (the waves of all its rows, key/value head by key/value head), then over the next ones, ... Where one begins is counted per key/value head.
// A sequence's row tile for the join: the first wave of its first result (of key/value head 0), how many results there are over its positions and how far
// apart, and how far key/value heads are; its first token, its first row among its sequence's, the sequence's rows. The first entry holds the number of
// them in `first`, and of the shared positions' results `parts`, `apart` and `waves`.
struct __attribute__((aligned(32))) TreeTile { int first, parts, apart, waves, t0, row0, rows; };

struct Draft {
    struct Seq {
        int t0, t1, len, rows, tiles, from, to, steps;
        __device__ __forceinline__ int waves() const { return (rows + 31) >> 5; }
    };
    // the shared positions' rows (every token) as a sequence of its own
    __device__ static __forceinline__ Seq of_shared(const TreeArgs &A) {
        Seq q = {0, 0, 0, A.a.shared ? att_start(A.a, A.a.nseq) * A.group : 0, 0, 0, A.a.shared, (A.a.shared + TREE_BN - 1) / TREE_BN};
        q.tiles = (q.rows + ATT_BM - 1) / ATT_BM;
        return q;
    }
    __device__ static __forceinline__ Seq of(const TreeArgs &A, int s) {
        const mmoe_attn_args &a = A.a;
        Seq q = {};
        if (s >= a.nseq) return q;
        // Whatever qstart and len hold, the rows lie inside the arrays and the positions inside the table: no difference here can wrap around (0 <= t0 <=
        // ntok, t1 >= t0, len >= 0)
        q.t0 = att_start(a, s); q.t1 = max(a.qstart[s + 1], q.t0); q.len = max(a.len[s], 0);
        const int n = q.t1 - q.t0, ctx = q.len - n;
        q.rows = min(min(q.t1, a.ntok) - q.t0, a.max_q) * A.group;
        q.tiles = (q.rows + ATT_BM - 1) / ATT_BM;
        q.from = a.shared;
        if (a.window > 0 && ctx > a.window) q.from = max(q.from, ctx - a.window);
        q.from &= ~(TREE_BN - 1);
        q.to = min(q.len - max(n - a.max_q, 0), a.max_len);
        q.steps = q.to > q.from ? (q.to - q.from + TREE_BN - 1) / TREE_BN : 0;
        return q;
    }
    // Pieces of a row tile: its steps times the pieces per step, rounded up (up to 2^-10 above a whole number that one is taken). Of two steps at
    // least, but for the shortest tiles: 12 results are joined in the time of 6 (26 tokens over 700 positions, 11 steps: 12.6 us, in 6 pieces 13.6; but 60 over
    // 3000: 48 pieces 19.6, 24 pieces 17.0)
    __device__ static __forceinline__ int cut(const Seq &q, float per) {
        return max(min((int)ceilf(fmaf((float)q.steps, per, -0x1p-10f)), max((q.steps + 1) >> 1, 12)), 1);
    }
    struct Mem { int sum[3][4], at[4]; };
    __device__ static __forceinline__ int wave_sum(int v) { return wave_reduce(v, [](int x, int y) { return x + y; }); }
    // Pieces per step; how many pieces there are, row tiles of the sequences and over the shared positions, waves of the latter, pieces of one of them (which
    // come first)
    struct Cut { float per; int pieces, own_tiles, shared_tiles, shared_waves, shared_k; };
    // The same for every thread of the workgroup (256). MANY: more than 64 sequences, else every wave does it by itself
    template <bool MANY> __device__ static __forceinline__ Cut plan(const TreeArgs &A, Mem &M) {
        const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, n = A.a.nseq;
        const Seq sh = of_shared(A), q = of(A, MANY ? tid : l);
        auto total = [&](auto &&f) {
            int v = f(q);
            if (!MANY) return wave_sum(v);
            for (int s = tid + 256; s < n; s += 256) v += f(of(A, s));
            v = wave_sum(v);
            __syncthreads();
            if (l == 0) M.sum[0][w] = v;
            __syncthreads();
            return M.sum[0][0] + M.sum[0][1] + M.sum[0][2] + M.sum[0][3];
        };
        Cut c;
        c.own_tiles = total([](const Seq &x) { return x.tiles; });
        c.shared_tiles = sh.tiles; c.shared_waves = sh.waves();
        const int all_tiles = sh.tiles + c.own_tiles;
        float per = 0.0f;
        int pieces = all_tiles;
        if (A.room) {
            // (the host has seen to it that all steps are a 32-bit number)
            const int steps = sh.tiles * sh.steps + total([](const Seq &x) { return x.tiles * x.steps; });
            // Up to as many row tiles as there is room for a search for pieces that fit at once. More of them take more rounds anyway: as long as a share of
            // the room makes them, which cuts the longest only, and no search. 20 tokens over 1500, 16 and 4 heads of 128 (128 pieces fit): 72 sequences 62
            // us and 120 85, without the search, in pieces half as large, 82 and 116; 200 sequences 145 us, in pieces half as large 177 (but 200 of 10 over 3000
            // with heads of 64: 165, 160)
            const bool few = all_tiles <= A.room;
            const int goal = A.room;
            // rounding up makes about half a piece more of each row tile
            per = fminf(((float)goal - (few ? 0.5f * (float)all_tiles : 0.0f)) / (float)max(steps, 1), 1.0f);
            for (int i = 0;; i++) {
                pieces = sh.tiles * cut(sh, per) + total([&](const Seq &x) { return x.tiles * cut(x, per); });
                if (!few || pieces <= goal) break;
                per = i < 6 ? per * fminf((float)goal / (float)pieces, 0.97f) : 0.0f;   // (at last each row tile one piece)
            }
        }
        if (pieces == 0 && A.room && blockIdx.x == 0 && tid == 0) A.tile_at[0] = {};   // the workspace may hold an earlier call's
        c.per = per; c.pieces = pieces; c.shared_k = cut(sh, per);
        return c;
    }
    // A piece: its sequence (-1: the shared positions), that one's first piece, first result and row tile, the pieces of its row tile
    struct Piece { int seq, base, result, tiles, k; Seq q; };
    template <bool MANY> __device__ static __forceinline__ bool piece(const TreeArgs &A, Mem &M, const Cut &c, int id, Piece &o) {
        const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, n = A.a.nseq, common = c.shared_tiles * c.shared_k, common_waves = c.shared_waves * c.shared_k;
        if (id < common) {
            o = {-1, 0, 0, 0, c.shared_k, of_shared(A)};
            return true;
        }
        // results are kept for row tiles that are cut, and for all with shared positions
        auto kept_of = [&](const Seq &x, int k) { return k > 1 || A.a.shared ? x.waves() * k : 0; };
        if (!MANY) {
            const Seq q = of(A, l);
            const int k = cut(q, c.per), mine = q.tiles * k;
            const int end = common + (int)scan_wave(mine), tiles = (int)scan_wave(q.tiles) - q.tiles;
            int result = 0;
            if (A.room) {   // (else every row tile is whole)
                const int kept = kept_of(q, k);
                result = common_waves + (int)scan_wave(kept) - kept;
            }
            const int s = __popcll(__ballot(id >= end));   // a prefix of the lanes
            if (s >= n) return false;
            auto lane = [&](int v) { return __builtin_amdgcn_readlane(v, s); };
            o.seq = s; o.base = lane(end - mine); o.result = lane(result); o.tiles = lane(tiles);
            o.q = {lane(q.t0), lane(q.t1), lane(q.len), lane(q.rows), lane(q.tiles), lane(q.from), lane(q.to), lane(q.steps)};
            o.k = cut(o.q, c.per);
            return true;
        }
        int before = common, tiles = 0, results = common_waves;
        if (tid == 0) M.at[0] = -1;
        for (int s0 = 0; s0 < n; s0 += 256) {
            const Seq x = of(A, s0 + tid);
            const int k = cut(x, c.per), mine = x.tiles * k, kept = kept_of(x, k);
            int end = (int)scan_wave(mine), t = (int)scan_wave(x.tiles), r = (int)scan_wave(kept);
            __syncthreads();   // the sums before have been read
            if (l == 63) { M.sum[0][w] = end; M.sum[1][w] = t; M.sum[2][w] = r; }
            __syncthreads();
            int ps = 0, ts = 0, rs = 0;
            for (int i = 0; i < 4; i++) {
                if (i < w) { end += M.sum[0][i]; t += M.sum[1][i]; r += M.sum[2][i]; }
                ps += M.sum[0][i]; ts += M.sum[1][i]; rs += M.sum[2][i];
            }
            end += before; t += tiles; r += results;
            if (id < end && id >= end - mine) { M.at[0] = s0 + tid; M.at[1] = end - mine; M.at[2] = t - x.tiles; M.at[3] = r - kept; }
            before += ps; tiles += ts; results += rs;
            if (id < before) break;
        }
        __syncthreads();
        o.seq = __builtin_amdgcn_readfirstlane(M.at[0]); o.base = __builtin_amdgcn_readfirstlane(M.at[1]); o.tiles = __builtin_amdgcn_readfirstlane(M.at[2]);
        o.result = __builtin_amdgcn_readfirstlane(M.at[3]);
        if (o.seq < 0) return false;
        o.q = of(A, o.seq);
        o.k = cut(o.q, c.per);
        return true;
    }
};

// For a row (a token and a query head) with ctx cached positions: out = sum over what it sees of softmax(scale q k + bias) v, lse the logarithm of the
// softmax's sum; the tile's two products, its masks and its running maximum are att_tile's, in 32 bits, weights rounded to the cache's type. A
// workgroup has one piece of one row tile of one key/value head. Not on LDS or registers but on the card's memory and on evenness it depends: every
// byte of the cache has to be read once (the row tiles of a sequence read it at the same time, from their die's cache), the pieces begin together and
// the last ends long after the median one. Measured with the join: 64 drafts of 10 to 40 tokens over 50 to 3000 positions, 16 and 4 heads of 128, 215 MB:
// 68 us, 3.2 TB/s (41 would be a copy's rate; pieces have 17 steps in the middle and 24 at most; begin 6 us, join 8); 4 drafts of 100 to 200 over 20000
// to 30000, capped: 168 to 184 us on several cards, 0.66 to 0.72 PFLOP/s, the matrix products beside three exponentials' work; 32 drafts of 64 in a window
// of 512: 24.6 us, whole row tiles, one wave per SIMD: 10 steps of 3450 cycles behind 14000 of dependent loads; 17 drafts behind 2048 shared positions,
// heads of 64 with slopes: 32.4 us, the exponentials and the sums beside them (seven and a half operations a score); one draft of 26 over 700: 12.7 us,
// latency.
// MANY: of more than 64 sequences most may be without tokens, so that there is a bound on the pieces far above their number: a workgroup takes more than
// one, one after the other, where there are more than the launch has workgroups.
template <int T, int D, bool CAP, bool BIAS, bool MANY>
__global__ void __launch_bounds__(256, 2) k_attn_tree(TreeArgs A) {
    __shared__ AttTileMem<D, TREE_BN> M;
    __shared__ Draft::Mem F;
    const Draft::Cut c = Draft::plan<MANY>(A, F);
    // Workgroups go to the card's dies in turn: each die a run of consecutive pieces, in which the row tiles of the same positions lie side by
    // side and read them from the die's own cache
    const int all = max(c.pieces, 0) * A.kv.heads, each = (all + 7) >> 3;
    for (int y = blockIdx.x >> 3; y < each; y += gridDim.x >> 3) {
        const int at = (int)(blockIdx.x & 7) * each + y, kvh = at / c.pieces, id = at - kvh * c.pieces;
        Draft::Piece o;
        if (at >= all || !Draft::piece<MANY>(A, F, c, id, o)) return;
        const Draft::Seq &q = o.q;
        const int k = __builtin_amdgcn_readfirstlane(o.k), steps = __builtin_amdgcn_readfirstlane(q.steps), i = (id - o.base) / q.tiles, tile = id - o.base - i * q.tiles;
        const bool whole = k == 1 && !A.a.shared;
        const int waves = q.waves(), first = tile * (ATT_BM / 32), result = o.result + i * waves;
        // (both fit if qstart ascends; if it does not, sums of what sequences claim may even have wrapped around)
        if ((whole || (result >= 0 && result + (int64_t)waves <= A.most_waves)) && (o.seq < 0 || (unsigned)(o.tiles + tile) < (unsigned)A.most_tiles)) {
            if (A.room && kvh == 0 && i == 0 && threadIdx.x == 0) {
                if (o.seq >= 0) A.tile_at[1 + o.tiles + tile] = {result * A.kv.heads + first, k, waves * A.kv.heads, waves, q.t0, tile * ATT_BM, q.rows};
                if (id == 0) A.tile_at[0] = {min(c.own_tiles, A.most_tiles), c.shared_k, c.shared_waves * A.kv.heads, c.shared_waves};
            }
            const int len = steps / k, more = steps - len * k;   // the first of them a step longer
            AttWork work = {};
            work.shared = o.seq < 0;
            work.at = {max(o.seq, 0), tile * ATT_BM, q.rows, q.t0};
            work.t1 = q.t1; work.len = q.len;
            work.kvh = kvh;
            work.p0 = q.from + (i * len + min(i, more)) * TREE_BN;
            work.p1 = min(work.p0 + (len + (i < more)) * TREE_BN, q.to);
            work.whole = whole;
            work.slot = (int64_t)result * A.kv.heads + kvh * waves + first;
            att_tile<T, D, CAP, BIAS, true>(tree_args(), work, M);
        }
        if (!MANY) return;
        __syncthreads();   // every wave is done with LDS
    }
}

// The partial results of a row tile put together, 32 rows by a workgroup: each result holds its weighted values, not yet divided, the maximum that its
// weights are counted from (in units of log 2) and their sum, with the sign set where results may not be finite. A lane has a row and 4 of each 8 dims,
// a wave a quarter of the dims; deep (few row tiles, so perhaps many results of each): a wave has a quarter of the results, a workgroup an eighth of
// the dims, and the waves join through LDS. The results come from memory (the pieces ran on other dies), so loads of eight results at once are what
// counts, and short code: a call's first instructions come from memory as well, and branches between the loads cost as much as the loads. Measured: 2.9
// to 4.1 us for one draft's 12 results, 8.5 us for 64 drafts (17 MB).
template <int T, int D, bool DEEP>
__global__ void __launch_bounds__(256) k_tree_join(TreeArgs A) {
    constexpr int C = DEEP ? D / 64 : D / 32, TJ_U = DEEP ? 8 : 512 / D;   // groups of 8 dims of a lane; results under way
    const mmoe_attn_args &a = A.a;
    __shared__ f4 acc[DEEP ? 3 : 1][C][64];
    __shared__ float2 stat[DEEP ? 3 : 1][32];
    const int l = threadIdx.x & 63, n = l & 31, hh = l >> 5, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned id = blockIdx.x;
    int share = wv;   // of the dims
    if (DEEP) { share = id & 7; id >>= 3; }
    const int w = id & 3;   // the tile's wave, its key/value head, its number
    id >>= 2;
    const int tile = (int)A.by_kv(id), kvh = id - tile * A.kv.heads;
    const TreeTile head_of = A.tile_at[0], t = A.tile_at[1 + tile];
    const int64_t first = t.first + kvh * (int64_t)t.waves + w, most = (int64_t)A.most_waves * A.kv.heads;
    const int r = t.row0 + w * 32 + n;
    const bool live = r < t.rows;
    const int row = min(r, t.rows - 1), j = (int)A.by_group(row), tok = t.t0 + j, head = kvh * A.group + row - j * A.group;
    // the results over the shared positions hold every token's rows
    const int common = a.shared ? head_of.parts : 0, rs = tok * A.group + row - j * A.group;
    const int64_t first_sh = kvh * (int64_t)head_of.waves + (rs >> 5);
    // None, or written by the piece that was all of it; nothing outside the arrays, whatever qstart holds (where it does not ascend, row tiles may be those of
    // an earlier call). One condition: the kernel's arguments are then asked for at once, not branch by branch.
    const bool some = (tile < head_of.first) & ((t.parts > 1) | (a.shared > 0)) & (t.parts > 0) & ((t.first | t.waves | t.apart | t.t0 | t.row0) >= 0) & (t.row0 + w * 32 < t.rows) &
                      (first + (t.parts - 1) * (int64_t)t.apart < most) & (t.rows <= (int64_t)(a.ntok - t.t0) * A.group);
    const bool some_sh = (a.shared == 0) | (((common | head_of.apart | head_of.waves) >= 0) & (first_sh + (common - 1) * (int64_t)head_of.apart < most));
    if (!some || !some_sh) return;
    const int parts = common + t.parts;
    const float2 *pm = A.pm + first * 32 + n, *pm_sh = A.pm + first_sh * 32 + (rs & 31);
    const f4 *po = (const f4 *)A.po + first * (8 * D) + 32 * hh + n, *po_sh = (const f4 *)A.po + first_sh * (8 * D) + 32 * hh + (rs & 31);
    struct Result { float2 v; f4 y[C]; };
    auto load = [&](Result &x, int p) {
        const bool c = p < common;
        const int64_t at = (c ? p * (int64_t)head_of.apart : (p - common) * (int64_t)t.apart) * 32;
        x.v = (c ? pm_sh : pm)[at];
        const f4 *q = (c ? po_sh : po) + at * (D / 4);
#pragma unroll
        for (int i = 0; i < C; i++) x.y[i] = q[(share * C + i) * 64];
    };
    float m = -__builtin_inff(), sum = 0.0f;
    f4 o[C] = {};
    bool wild = false;
    // N results more: no branches, so that the code is short (a call's first instructions come from memory, too)
    auto add = [&](const Result *x, auto n) {
        float mn = m;
#pragma unroll
        for (int u = 0; u < n.value; u++) mn = fmaxf(mn, x[u].v.y != 0.0f ? x[u].v.x : -__builtin_inff());
        const float by = mn == -__builtin_inff() ? 0.0f : mn, al = exp2_(m - by);
        m = mn; sum *= al;
#pragma unroll
        for (int c = 0; c < C; c++) o[c] *= al;
#pragma unroll
        for (int u = 0; u < n.value; u++) {
            const float e = x[u].v.y != 0.0f ? exp2_(x[u].v.x - by) : 0.0f;
            sum = fmaf(fabsf(x[u].v.y), e, sum);
            wild |= __float_as_int(x[u].v.y) < 0;   // (a sum of 0 has a sign, too)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[c][i] = fmaf(e, x[u].y[c][i], o[c][i]);
        }
    };
    constexpr int STEP = DEEP ? 4 : 1;
#pragma unroll 1
    for (int p0 = DEEP ? wv : 0; p0 < parts; p0 += TJ_U * STEP) {
        Result x[TJ_U];
#pragma unroll
        for (int u = 0; u < TJ_U; u++) {
            x[u] = {};
            if (p0 + u * STEP < parts) load(x[u], p0 + u * STEP);
        }
        add(x, std::integral_constant<int, TJ_U>{});
    }
    if (DEEP) {
        if (wv) {
#pragma unroll
            for (int c = 0; c < C; c++) acc[wv - 1][c][l] = o[c];
            if (hh == 0) stat[wv - 1][n] = make_float2(m, wild ? -sum : sum);
        }
        __syncthreads();
        if (wv) return;
        Result x[3];
#pragma unroll
        for (int i = 0; i < 3; i++) {
            x[i].v = stat[i][n];
#pragma unroll
            for (int c = 0; c < C; c++) x[i].y[c] = acc[i][c][l];
        }
        add(x, std::integral_constant<int, 3>{});
    }
    if (__any(wild && live)) {   // once more: results that are not finite count whatever their weight, and where every score was -inf
#pragma unroll
        for (int c = 0; c < C; c++) o[c] = f4{0, 0, 0, 0};
#pragma unroll 1
        for (int p = 0; p < parts; p++) {
            Result x;
            load(x, p);
            const float e = x.v.y != 0.0f ? exp2_(x.v.x - m) : 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[c][i] = e != 0.0f ? fmaf(e, x.y[c][i], o[c][i]) : o[c][i] + only_odd(x.y[c][i]);
        }
    }
    if (!live) return;
    const float inv = 1.0f / sum;
    uint16_t *out = (uint16_t *)a.out + (int64_t)tok * a.out_token + head * a.out_head + share * (8 * C) + 4 * hh;
#pragma unroll
    for (int c = 0; c < C; c++) {
        uint2 v = make_uint2(pack2<T>(o[c][0] * inv, o[c][1] * inv), pack2<T>(o[c][2] * inv, o[c][3] * inv));
        if (sum == 0.0f) v = make_uint2(0, 0);
        *(uint2 *)(out + 8 * c) = v;
    }
    if (a.lse && share == 0 && hh == 0) a.lse[(int64_t)tok * a.heads + head] = sum == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(sum)) * ATT_LN2;
}

