// K7: attention of one new token per request over a KV cache of pages.
//
// The ordinary decode step beside the tree verification of K2 (what the
// reference's autoregressive loop, cast_trees/decode.py:211-231, leaves to
// the model's attention): request b's query sees the keys of slots
// [start, len), len = seq_len[b], start = len - window where a window is set,
//   o = sum_t softmax_t(f(scale q . k_t)) v_t,   f(s) = cap tanh(s / cap)
// with a cap, the identity without.  Slot t lies in page
// table[b][t / page_size] at offset t % page_size.  Query head h reads KV head
// h / (Hq / Hkv).
//
// Bound by the K and V bytes: 4 D bytes a key and KV head in 16 bits against
// 4 D G flops.  The G query heads of a KV head are the columns of 16-wide
// matrix products, so each key is read once for all of them and the products
// cost a tenth of the time its bytes take.
//
// A work item is a run of key tiles of one (request, KV head, block of 16 query
// heads); the four waves of a workgroup take 16 KB of keys in turn, each on its own with its
// own running maximum and sum, and join through LDS at the end.  No operand
// goes through LDS:
//   S^T = K Q^T   the operand's lane (key, g) wants chunks 4 c + g of its key's
//                 row, 64 bytes of 16 rows at a time; loaded like that, every
//                 128-byte line is asked for twice.  A load takes 128 bytes of
//                 8 rows instead, and a DPP move a register trades the halves
//                 of two of them;
//   O^T += V^T P^T  a lane holds D/16 elements of 8 keys (16-byte chunks,
//                 neighbouring lanes reading neighbouring chunks of a row),
//                 which v_perm turns into 8 keys of each element; the keys it
//                 takes are those whose weights the first product left in its
//                 registers, and the order of the head dim over the operand's
//                 rows is free.
// fp32 runs both products on the fp32 matrix instruction.  16-bit weights are
// two terms (p - round(p) is the second), so that they keep float precision
// where the matrix pipes have room; V rows of masked keys are zeroed, as
// memory behind the last token may hold anything.
//
// The next tile's loads are issued before the current one is used; page ids
// are loaded a group of tiles ahead.  The keys of all requests are dealt out in
// equal runs, pieces of a request write (O, max, sum) in float and a second
// kernel joins them.  Measured (8 KV and 32 query heads of 128, bf16): 8
// requests of 8k keys 43.5 us = 6.2 TB/s and 4.5 us of join, 64 of 300 to 8k
// 208 us = 6.0 TB/s and 5 us; a large read alone reaches 6.0 to 6.3 TB/s.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <mutex>

#include "cast_common.hpp"

namespace cast {

constexpr float kPLn2 = 0.69314718055994530942f;
constexpr float kPLog2e = 1.44269504088896340736f;
constexpr int kPWaves = 4;
// What a piece costs beside its tiles, in tiles of 32 KB (head dim 64) and of
// 64 KB and more (measured before units that cannot be long were left whole): 200 requests of up to 1k keys at D = 64, fp16, 43.3, 36.5, 35.2
// and 35.9 us for 0 to 3; 64 of 300 to 8k at D = 128, bf16, 219.5, 222, 225, 230.
constexpr int piece_cost(int D) { return D == 64 ? 2 : 1; }
constexpr int kLensLds = 1024;           // batches whose lengths a workgroup keeps in LDS for its schedule
// Fewest key tiles of a piece, unless the caller says: one request of 2k keys
// over 8 KV heads 8.9, 10.8, 12.3 and 16.4 us (without the join) at 1, 2, 4, 8.
constexpr int kMinTiles = 1;
// Tiles a workgroup should have before a CU gets a second one, where units are
// fewer than CUs: one request of 32k keys 24.1 + 4.0 us (attention, join) on 256
// workgroups of 8 tiles, 24.8 + 5.0 on 512 of 4.  (Units of their own are better
// spread: 200 requests of up to 1k keys, 4 KV heads, scheduled: 35 us on 768, 37.6 on 440.)
constexpr int kFewTiles = 8;

struct PagedAttnArgs {
    const void *q, *k, *v;
    void *out;
    float *lse;
    const int32_t *table, *seq_len;
    int32_t *status;
    int64_t table_ld, q_req, q_head, o_req, o_head;                      // elements (q, out)
    int64_t kp_page, kp_head, kp_tok, vp_page, vp_head, vp_tok;          // bytes
    int32_t n_pages, page_size, batch, Hq, Hkv, G, rbs, D, cap, window;  // cap: slots a table row covers
    FastDiv by_page;    // division by page_size
    int32_t wgs;        // workgroups of the attention kernel
    int32_t cus;        // CUs of the device
    int32_t least;      // fewest tiles of a piece; 0: one workgroup per unit, no pieces
    int32_t cut;        // pieces of exactly `least` tiles, as the caller says
    int32_t prows;      // rows of a partial: min(16, G)
    float scale, softcap;   // scale: natural scale (softcap) or times log2(e)
    int32_t *units;     // workspace: [units][2], a unit's first partial slot and how many pieces it has (1: none, it is out)
    float *part_ml;     // [2 wgs][prows][2] running maximum (base 2) and sum; sum < 0: a page id is bad
    float *part_o;      // [2 wgs][prows][D]
};

// ---- lanes and waves
__device__ __forceinline__ int p_wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
__device__ __forceinline__ int p_wave_sum(int x) { return __builtin_amdgcn_readlane(p_wave_scan(x), 63); }

// The largest / the sum over the four lanes that share l16 = lane % 16.
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// The cache policy of loads that this kernel does once: not kept in the caches (the nt bit).
constexpr int kOnce = 2;

// ---- formats
struct PF32 {
    static constexpr int kBytes = 4, kBlocks = 1;     // 16-key blocks per wave tile
    static constexpr float kPScale = 1.f;
    using T = float;
};
struct PBf16 : Bf16 {
    static constexpr int kBytes = 2, kBlocks = 2;
    static constexpr float kPScale = 1.f;
    using T = uint16_t;
    static __device__ __forceinline__ floatx4 mma16(vec8 a, vec8 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
// fp16 weights are scaled by 2^15, so that their second term stays a normal
// number (weights are at most 1).
struct PFp16 : Fp16 {
    static constexpr int kBytes = 2, kBlocks = 2;
    static constexpr float kPScale = 32768.f;
    using T = uint16_t;
    static __device__ __forceinline__ floatx4 mma16(vec8 a, vec8 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// ---- the schedule, found by every workgroup from the lengths.  A unit
// (request, block of 16 query heads, KV head) is a run of key tiles.
//  - Cut: every unit into equal pieces of at most c tiles, a workgroup each,
//    where c is an even share of all tiles (or 9/8 of it) and the pieces are no
//    more than the workgroups that the device holds.
//  - Stretches, where they would be more: the units lie in a line, piece_cost
//    empty places (what a piece costs beside its tiles) and then a place per
//    tile each, and the workgroups take equal stretches of it (with `all`
//    places and W workgroups, the first all % W take one more than the others).
//    A workgroup walks its stretch unit by unit; it meets at most two units
//    that it does not cover whole, its first and its last.
// A unit that a workgroup covers whole goes to the output, a piece of one to a
// partial, two slots a workgroup.  Measured, one against the other: 8 requests
// whose windows take 32 or 33 tiles, D = 256, cut 55.1 us, stretches 59.2 (a
// second piece costs a join and a pipeline's start); 64 requests of 300 to 8k
// keys cut 250 us, stretches 222 (the cut ran in one and a half rounds).
struct PagedReq {
    int start, len, t0, tiles;   // visible slots [start, len), key tiles [t0, t0 + tiles); a tile where none is seen
};
__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs &a, int tk, int len) {
    PagedReq r{0, 0, 0, 1};
    if (len <= 0 || len > a.cap) return r;
    r.len = len;
    r.start = a.window > 0 && len > a.window ? len - a.window : 0;
    r.t0 = r.start / tk;
    r.tiles = (len + tk - 1) / tk - r.t0;
    return r;
}
__device__ __forceinline__ int splits_of(int tiles, int c) {
    return tiles <= c ? 1 : (int)(((uint32_t)tiles + (uint32_t)c - 1) / (uint32_t)c);
}
struct Stretches {
    int W, q, r;
    __device__ __forceinline__ Stretches(int wgs, int least, int all) {
        W = min(wgs, (int)(((uint32_t)all + (uint32_t)least - 1) / (uint32_t)least));
        q = (int)((uint32_t)all / (uint32_t)W);
        r = all - q * W;
    }
    __device__ __forceinline__ int first(int x) const { return x * q + min(x, r); }   // workgroup x's first place
    __device__ __forceinline__ int of(int at) const {                                 // whose place it is
        const int wide = r * (q + 1);
        return at < wide ? (int)((uint32_t)at / (uint32_t)(q + 1)) : r + (int)((uint32_t)(at - wide) / (uint32_t)q);
    }
};

template <int D, typename E, bool PAD, bool ANY>
__global__ __launch_bounds__(kPWaves * 64) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : (D == 128 ? 2 : 3) - ANY)))
void paged_attn_kernel(PagedAttnArgs a) {
    using T = typename E::T;
    constexpr bool F32 = E::kBytes == 4;
    constexpr int KB = E::kBlocks;                 // 16-key blocks of a wave's tile
    constexpr int WK = 16 * KB;                    // keys of a wave's tile
    constexpr int TK = WK * kPWaves;               // keys of a workgroup's tile
    constexpr int KC = F32 ? D / 16 : D / 32;      // 16-byte chunks of K a lane holds
    constexpr int KE = 16 / E::kBytes;             // elements of such a chunk
    constexpr int EPC = F32 || D == 64 ? 4 : 8;    // elements of a V chunk
    constexpr int VC = D / (16 * EPC);             // V chunks of a key a lane holds
    constexpr int VK = 4 * KB;                     // keys a lane holds V of
    constexpr int NA = D / 16;                     // 16-row blocks of O^T
    constexpr bool kAhead = !(ANY && F32 && D == 256);   // two tiles in flight (here they, and 64-bit addresses, spill)
    constexpr int OP = D + 4;                      // row stride of the join's O (floats)
    __shared__ __attribute__((aligned(16))) float Os[kPWaves][16][OP];
    __shared__ float ML[kPWaves][16][2];
    __shared__ int Lens[kLensLds];

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, l8 = lane & 7, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int dr = PAD ? a.D : D;

    // ---- this workgroup's places [p, p_end) of the line of units, in which
    // request b's start at `base`; a unit is `cost` empty places and its tiles
    const int per = a.Hkv * a.rbs, x = blockIdx.x;
    int b0 = 0, b = 0, base = 0, p = 0, p_first = 0, p_end = 0, len_l = 0, cost = 0;
    if (a.least) {
        // (loops of little code: what runs once waits for its instructions)
        const int *lens = a.seq_len;
        if (a.batch <= kLensLds) {
            for (int i = tid; i < a.batch; i += kPWaves * 64) Lens[i] = a.seq_len[i];
            __syncthreads();
            lens = Lens;
        }
        // the places of this lane's request in the block of 64 from k on, or
        // its units' pieces of up to c tiles
        auto count = [&](int k, int c) __attribute__((always_inline)) {
            len_l = lens[min(k + lane, a.batch - 1)];
            const int n = paged_req(a, TK, len_l).tiles;
            return k + lane >= a.batch ? 0 : (c ? splits_of(n, c) : n + piece_cost(D)) * per;
        };
        int all = 0, c = a.cut ? a.least : 0, items = 0, wgs = a.wgs;
        for (;;) {
            int n = 0;
#pragma unroll 1
            for (int k = 0; k < a.batch; k += 64) n += p_wave_sum(count(k, c));
            if (a.cut) {
                items = n;
                break;
            }
            if (c == 0) {
                all = n;
                const int tiles = all - a.batch * per * piece_cost(D);
                if (a.batch * per < a.cus) wgs = min(wgs, max(a.cus, tiles / kFewTiles));
                c = max(a.least, (int)(((uint32_t)tiles + (uint32_t)wgs - 1) / (uint32_t)wgs));
                if (a.batch * per > a.wgs) {   // (a piece per unit is too many)
                    c = 0;
                    break;
                }
            } else if (n <= a.wgs) {
                items = n;
                break;
            } else if (items || c < 8) {
                items = c = 0;
                break;
            } else {
                items = n;
                c += c >> 3;
            }
        }
        const Stretches st(wgs, a.least, c ? a.least : all);
        if (x >= (c ? items : st.W)) return;
        const int at = c ? x : st.first(x);
#pragma unroll 1
        for (int k = 0; k < a.batch; k += 64) {
            const int n = count(k, c), incl = p_wave_scan(n);
            const uint64_t past = __ballot(base + incl <= at);
            b0 = k;
            if (~past) {
                const int j = __builtin_ctzll(~past);
                b = k + j;
                base += __builtin_amdgcn_readlane(incl - n, j);
                break;
            }
            base += __builtin_amdgcn_readlane(incl, 63);
        }
        if (x == 0 && w == 0)
            for (int k = lane; k < a.batch; k += 64)
                if (lens[k] < 0 || lens[k] > a.cap) raise_flag(a.status, CAST_FLAG_BAD_OFFSETS);
        if (c) {
            const int tiles = paged_req(a, TK, __builtin_amdgcn_readlane(len_l, b - b0)).tiles, ns = splits_of(tiles, c);
            const int unit = (int)((uint32_t)(x - base) / (uint32_t)ns), s = x - base - unit * ns;
            if (s == 0 && tid == 0) {
                a.units[2 * (b * per + unit)] = 2 * x;
                a.units[2 * (b * per + unit) + 1] = ns;
            }
            base = 0;
            p = unit * tiles + (int)((int64_t)tiles * s / ns);
            p_end = unit * tiles + (int)((int64_t)tiles * (s + 1) / ns);
        } else {
            cost = piece_cost(D);
            p = at;
            p_end = st.first(x + 1);
            // the units whose first tile lies in the stretch: a lane each
            if (w == 0) {
                int bb = b, from = base;
                for (int left = p; left < p_end; ++bb) {
                    const int tiles = paged_req(a, TK, lens[bb]).tiles;
                    for (int u = lane; u < per; u += 64) {
                        const int unit = from + u * (tiles + cost), first = unit + cost;
                        if (first >= p && first < p_end) {
                            // (a stretch that starts in front of the unit has a piece of the one before)
                            a.units[2 * (bb * per + u)] = 2 * x + (p < unit);
                            a.units[2 * (bb * per + u) + 1] = st.of(first + tiles - 1) - x + 1;
                        }
                    }
                    left = from += (tiles + cost) * per;
                }
            }
            // on to its first tile
            const int width = paged_req(a, TK, __builtin_amdgcn_readlane(len_l, b - b0)).tiles + cost;
            const int in = (int)((uint32_t)(p - base) % (uint32_t)width);
            if (in < cost) p += cost - in;
            if (p >= p_end) return;
        }
        p_first = p;
    } else {
        b = (int)((uint32_t)x / (uint32_t)per);
        b0 = b;
        len_l = a.seq_len[b];
        const int tiles = paged_req(a, TK, __builtin_amdgcn_readfirstlane(len_l)).tiles;
        p_first = p = (x - b * per) * tiles;
        p_end = p + tiles;
        if (x == b * per && tid == 0 && (len_l < 0 || len_l > a.cap)) raise_flag(a.status, CAST_FLAG_BAD_OFFSETS);
    }
    // (wave-uniform all along; told so, that branches and addresses are scalar)
    auto uni = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(v); };
    p = uni(p), p_first = uni(p_first), p_end = uni(p_end), base = uni(base), b = uni(b), b0 = uni(b0);
    // lane j of a wave knows the length of request b0 + j
    auto lengths = [&](int from) __attribute__((always_inline)) {
        b0 = from;
        len_l = a.seq_len[min(from + lane, a.batch - 1)];
    };
    // The piece of the line at place p, a tile of request b, whose places start
    // at `base`.
    struct Piece {
        int b, h, rb, start, len;   // visible slots [start, len)
        int key0, nt;               // the wave's first key, tiles
        bool whole, last;           // all of its unit, up to its end
    };
    auto piece = [&](int p, int b, int base) __attribute__((always_inline)) {
        const PagedReq rq = paged_req(a, TK, __builtin_amdgcn_readlane(len_l, b - b0));
        const int width = rq.tiles + cost, unit = (int)((uint32_t)(p - base) / (uint32_t)width);
        const int ta = p - base - unit * width - cost;
        Piece c;
        c.b = b;
        c.rb = unit / a.Hkv;
        c.h = unit - c.rb * a.Hkv;
        c.start = rq.start;
        c.len = rq.len;
        c.key0 = (rq.t0 + ta) * TK + w * WK;
        c.nt = min(p_end - p, rq.tiles - ta);
        c.whole = c.nt == rq.tiles;
        c.last = c.nt == rq.tiles - ta;
        return c;
    };

    // ---- Q^T: head l16 of the piece's block, chunks as K's
    uint32_t qraw[KC][4];
    auto load_q = [&](const Piece &c) __attribute__((always_inline)) {
        const T *qp = static_cast<const T *>(a.q) + (int64_t)c.b * a.q_req + (int64_t)(c.h * a.G + c.rb * 16 + l16) * a.q_head;
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const int d = F32 ? k * 16 + g * 4 : k * 32 + g * 8;
            const bool in = l16 < a.G - c.rb * 16 && (!PAD || d < dr);
            const u32x4 y = in ? *reinterpret_cast<const u32x4 *>(qp + d) : u32x4{};
#pragma unroll
            for (int i = 0; i < 4; ++i) qraw[k][i] = y[i];
        }
    };

    // ---- page ids, kGroup tiles of them in the lanes of a register: without
    // ANY, where a 16-key block lies within one page, one a block, with it one a
    // key; the next group's are loaded a group ahead.
    constexpr int kIds = ANY ? WK : KB, kGroup = 64 / kIds;
    auto seen = [&](const Piece &c, int key) __attribute__((always_inline)) { return min(max(key, c.start), c.len - 1); };
    auto load_ids = [&](const Piece &c, int i0, bool &bad) __attribute__((always_inline)) {   // of the group at tile i0
        if (i0 >= c.nt || c.len == 0) return 0;
        const int i = min(i0 + lane / kIds, c.nt - 1);
        const int key = seen(c, c.key0 + i * TK + lane % kIds * (WK / kIds));
        const int id = a.table[(int64_t)c.b * a.table_ld + a.by_page.div(key)];
        bad |= id < 0 || id >= a.n_pages;
        return min(max(id, 0), a.n_pages - 1);   // always a page of the pool
    };

    struct Tile {
        u32x4 k[KB][KC];
        uint32_t v[VK][VC][EPC * E::kBytes / 4];
    };
    constexpr int VW = EPC * E::kBytes / 4;        // 32-bit words of a V chunk
    // Byte offsets of this lane's chunks within a 16-key block.  Without ANY
    // they belong to a buffer resource that ends behind the block's last seen
    // key: what lies past it, and past the head dim, loads as zeros.
    constexpr uint32_t kNowhere = 0x7ffffff0u;
    auto k_at = [&](int c) __attribute__((always_inline)) {
        const int d = ((c >> 1) * 8 + (l16 >> 3) * 4 + g) * KE;
        return PAD && d >= dr ? kNowhere : (uint32_t)(8 * (c & 1) + l8) * (uint32_t)a.kp_tok + (uint32_t)(d * E::kBytes);
    };
    auto v_at = [&](int r, int c) __attribute__((always_inline)) {
        const int d = (c * 16 + l16) * EPC;
        return PAD && d >= dr ? kNowhere : (uint32_t)(4 * g + r) * (uint32_t)a.vp_tok + (uint32_t)(d * E::kBytes);
    };
    auto block = [&](const char *from, int keys, int64_t tok) __attribute__((always_inline)) {
        const int bytes = keys > 0 ? (min(keys, 16) - 1) * (int)tok + dr * E::kBytes : 0;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(from), 0, bytes, 0x00020000);
    };
    auto set_v = [&](Tile &t, int j, int c, auto y) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < VW; ++e) t.v[j][c][e] = y[e];
    };
    // tile i of the piece, its ids in `ids`
    auto load_tile = [&](Tile &t, const Piece &cur, int i, int ids) __attribute__((always_inline)) {
        if (ANY && (cur.len == 0 || i >= cur.nt)) return;
        const char *kbase = static_cast<const char *>(a.k) + (int64_t)cur.h * a.kp_head;
        const char *vbase = static_cast<const char *>(a.v) + (int64_t)cur.h * a.vp_head;
        const int kt = cur.key0 + i * TK;
#pragma unroll
        for (int t16 = 0; t16 < KB; ++t16) {
            const int kb = kt + 16 * t16;
            if constexpr (!ANY) {
                // the block's seen keys share a page
                // (no branch: a tile past the piece's last is a load of nothing)
                const int kc = max(seen(cur, kb), 0), off = kb - a.by_page.div(kc) * a.page_size;
                const int keys = i < cur.nt && kb + 16 > cur.start ? cur.len - kb : 0;
                const int64_t id = __builtin_amdgcn_readlane(ids, i % kGroup * KB + t16);
                const __amdgpu_buffer_rsrc_t kr = block(kbase + id * a.kp_page + off * a.kp_tok, keys, a.kp_tok);
                const __amdgpu_buffer_rsrc_t vr = block(vbase + id * a.vp_page + off * a.vp_tok, keys, a.vp_tok);
#pragma unroll
                for (int c = 0; c < KC; ++c)
                    t.k[t16][c] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, (int)k_at(c), 0, kOnce));
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        if constexpr (VW == 4)
                            set_v(t, 4 * t16 + r, c, __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, (int)v_at(r, c), 0, kOnce)));
                        else
                            set_v(t, 4 * t16 + r, c, __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vr, (int)v_at(r, c), 0, kOnce)));
                    }
            } else {
                // every key's own page; keys that are not seen are clamped into those that are
                auto row_at = [&](const char *pool, int64_t page, int64_t tok, int in) __attribute__((always_inline)) {
                    const int key = seen(cur, kb + in), off = key - a.by_page.div(key) * a.page_size;
                    return pool + (int64_t)__shfl(ids, i % kGroup * WK + 16 * t16 + in) * page + (int64_t)off * tok;
                };
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const char *kp = row_at(kbase, a.kp_page, a.kp_tok, 8 * y + l8);
#pragma unroll
                    for (int c = y; c < KC; c += 2) {
                        const int d = ((c >> 1) * 8 + (l16 >> 3) * 4 + g) * KE;
                        t.k[t16][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kp + min(d, dr - KE) * E::kBytes));
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const char *vp = row_at(vbase, a.vp_page, a.vp_tok, 4 * g + r);
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        const char *from = vp + min((c * 16 + l16) * EPC, dr - EPC) * E::kBytes;
                        if constexpr (VW == 4)
                            set_v(t, 4 * t16 + r, c, __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from)));
                        else
                            set_v(t, 4 * t16 + r, c, __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(from)));
                    }
                }
            }
        }
    };

    // a score's base-2 exponent is the product (capped: the tanh) times to_log2
    const float inv_cap = a.softcap > 0.f ? fminf(a.scale / a.softcap, 0x1.fffffep127f) : 0.f;
    const float to_log2 = a.softcap > 0.f ? a.softcap * kPLog2e : a.scale;
    floatx4 acc[NA];
    float m, l;
    bool again;   // see below
    auto use_tile = [&](Tile &t, const Piece &cur, int i) __attribute__((always_inline)) {
        const int kt = cur.key0 + i * TK;
        const bool edge = kt < cur.start || kt + WK > cur.len;
        float p[KB][4];
        __builtin_amdgcn_sched_barrier(0);   // (in this order: a tile's registers, not two stages')
        // ---- scores, scaled where their exponent is taken (one rounding)
#pragma unroll
        for (int t16 = 0; t16 < KB; ++t16) {
            // (fp32: two sums of every second product, half the roundings and half the wait)
            constexpr int NS = F32 ? 2 : 1;
            floatx4 sum[NS];
#pragma unroll
            for (int e = 0; e < NS; ++e) sum[e] = floatx4{};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                // words of chunk pair (c & ~1, c | 1): the loads left the first
                // eight keys in one register, the others in the next
                u32x4 kx;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t near = t.k[t16][c & ~1][e], far = t.k[t16][c | 1][e];
                    kx[e] = c & 1 ? (uint32_t)__builtin_amdgcn_update_dpp((int)far, (int)near, 0x128, 0xf, 0x3, false)
                                  : (uint32_t)__builtin_amdgcn_update_dpp((int)near, (int)far, 0x128, 0xf, 0xc, false);
                }
                if constexpr (ANY) {
                    // (chunks past the head dim were read from its last one)
                    if ((F32 ? c * 16 + g * 4 : c * 32 + g * 8) >= dr) kx = u32x4{};
                }
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t kw = kx[e];   // (a bit cast of the element itself reads element 0)
                        sum[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kw),
                                                                          __builtin_bit_cast(float, qraw[c][e]), sum[e & 1], 0, 0, 0);
                    }
                } else {
                    const u32x4 qx = {qraw[c][0], qraw[c][1], qraw[c][2], qraw[c][3]};
                    sum[0] = E::mma16(__builtin_bit_cast(typename E::vec8, kx), __builtin_bit_cast(typename E::vec8, qx), sum[0]);
                }
            }
            floatx4 s4 = sum[0];
            if constexpr (F32) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s4[r] = sum[0][r] + sum[1][r];
            }
            if (a.softcap > 0.f) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // tanh: 1 - 2 / (e^2x + 1), near 0 (where that cancels) its
                    // series to x^9, within 1e-8 of the value up to 1/4
                    const float x = s4[r] * inv_cap, x2 = x * x;
                    const float far = 1.f - 2.f / (__builtin_amdgcn_exp2f(x * (2.f * kPLog2e)) + 1.f);
                    const float poly = fmaf(fmaf(fmaf(62.f / 2835.f, x2, -17.f / 315.f), x2, 2.f / 15.f), x2, -1.f / 3.f);
                    const float near = fmaf(x * x2, poly, x);
                    p[t16][r] = x2 < 0.0625f ? near : far;
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) p[t16][r] = s4[r];
            }
        }
        if (edge) {
#pragma unroll
            for (int t16 = 0; t16 < KB; ++t16)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = kt + 16 * t16 + 4 * g + r;
                    if (key < cur.start || key >= cur.len) {
                        p[t16][r] = -INFINITY;
                        // (rows past the last key were loaded as zeros)
                        if (ANY || key < cur.start) {
#pragma unroll
                            for (int c = 0; c < VC; ++c)
#pragma unroll
                                for (int e = 0; e < VW; ++e) t.v[4 * t16 + r][c][e] = 0u;
                        }
                    }
                }
        }
        // ---- running maximum (base 2): moved for all columns at once, when any needs it
        float top = p[0][0];
#pragma unroll
        for (int t16 = 0; t16 < KB; ++t16)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, p[t16][r]);
        if (__any(top * to_log2 > m)) {
            const float mn = fmaxf(m, quad_max(top) * to_log2);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int n = 0; n < NA; ++n) acc[n] *= alpha;
        }
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int t16 = 0; t16 < KB; ++t16)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[t16][r] = __builtin_amdgcn_exp2f(fmaf(p[t16][r], to_log2, -ms));
                l += p[t16][r];
            }
        // ---- O^T += V^T P^T
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (F32) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int e = 0; e < EPC; ++e)
                        acc[c * EPC + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, t.v[r][c][e]), p[0][r],
                                                                                acc[c * EPC + e], 0, 0, 0);
        } else {
            u32x4 hi, lo;
#pragma unroll
            for (int t16 = 0; t16 < 2; ++t16)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float x = p[t16][r] * E::kPScale, y = p[t16][r + 1] * E::kPScale;
                    const uint32_t top2 = E::pack2(x, y);
                    hi[2 * t16 + r / 2] = top2;
                    lo[2 * t16 + r / 2] = E::pack2(x - E::widen((uint16_t)top2), y - E::widen((uint16_t)(top2 >> 16)));
                }
            if (again) {
                // weights of one sign, none rounded to zero: infinities keep theirs
#pragma unroll
                for (int t16 = 0; t16 < 2; ++t16)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const float x = p[t16][r], y = p[t16][r + 1];
                        hi[2 * t16 + r / 2] = E::pack2(x > 0.f ? fmaxf(x, 0x1p-14f) : x, y > 0.f ? fmaxf(y, 0x1p-14f) : y);
                    }
                lo = hi;
            }
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int e = 0; e < EPC; ++e) {
                    const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
                    u32x4 vx;
#pragma unroll
                    for (int j = 0; j < 4; ++j) vx[j] = __builtin_amdgcn_perm(t.v[2 * j + 1][c][e / 2], t.v[2 * j][c][e / 2], sel);
                    const auto vv = __builtin_bit_cast(typename E::vec8, vx);
                    acc[c * EPC + e] = E::mma16(vv, __builtin_bit_cast(typename E::vec8, hi), acc[c * EPC + e]);
                    acc[c * EPC + e] = E::mma16(vv, __builtin_bit_cast(typename E::vec8, lo), acc[c * EPC + e]);
                    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
        }
    };

    // where the wave's O^T lies in its part of the join's LDS
    auto place = [&](int c, int r) __attribute__((always_inline)) { return &Os[w][l16][(c * 16 + 4 * g + r) * EPC]; };
    // ---- piece by piece: the next one's page ids are loaded when one begins,
    // its first tile and Q before the one's join, whose LDS round trip they
    // run beside
    Tile even;
    bool bad = false;
    Piece cur = piece(p, b, base);
    int ids = load_ids(cur, 0, bad), ahead = load_ids(cur, kGroup, bad);
    load_q(cur);
    if (!ANY) load_tile(even, cur, 0, ids);
    for (;;) {
    if (ANY) load_tile(even, cur, 0, ids);
    const int p_next = uni(p + cur.nt + (cur.last ? cost : 0));
    const bool more = p_next < p_end;
    bool bad_next = false;
    int ids_next = 0, ahead_next = 0;
    if (more) {
        const int after = base + (paged_req(a, TK, __builtin_amdgcn_readlane(len_l, b - b0)).tiles + cost) * per;
        if (p_next >= after) {
            base = after;
            if (++b == b0 + 64) lengths(b);
        }
        const Piece next = piece(p_next, b, base);
        ids_next = load_ids(next, 0, bad_next);
        ahead_next = load_ids(next, kGroup, bad_next);
    }
#pragma unroll
    for (int n = 0; n < NA; ++n) acc[n] = floatx4{};
    m = -INFINITY;
    l = 0.f;
    again = false;
    const int rows = min(16, a.G - cur.rb * 16);   // query heads of this block
    if (cur.len > 0) {
        for (;;) {
            if constexpr (!kAhead) {
                for (int i = 0;;) {
                    use_tile(even, cur, i);
                    if (++i >= cur.nt) break;
                    if (i % kGroup == 0) ids = ahead, ahead = load_ids(cur, i + kGroup, bad);
                    load_tile(even, cur, i, ids);
                }
            }
            for (int i = kAhead ? 0 : cur.nt; i < cur.nt; i += 2) {
                Tile odd;
                load_tile(odd, cur, i + 1, ids);
                use_tile(even, cur, i);
                if (i + 1 >= cur.nt) break;
                if ((i + 2) % kGroup == 0) ids = ahead, ahead = load_ids(cur, i + 2 + kGroup, bad);
                load_tile(even, cur, i + 2, ids);
                use_tile(odd, cur, i + 1);
            }
            if (F32 || again) break;
            // An infinite V times a weight's second term, of either sign or
            // zero, is no number where infinity is meant: a wave whose sums
            // are not all finite walks its keys again with weights of one
            // sign, which decide only the elements that were not finite.
            float z = 0.f;
#pragma unroll
            for (int n = 0; n < NA; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) z = fmaf(acc[n][r], 0.f, z);
            if (!__any(l16 < rows && !(z == 0.f))) break;
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < EPC; ++e) {
                        place(c, r)[e] = acc[c * EPC + e][r];
                        acc[c * EPC + e][r] = 0.f;
                    }
            m = -INFINITY;
            l = 0.f;
            again = true;
            ids = load_ids(cur, 0, bad), ahead = load_ids(cur, kGroup, bad);
            load_tile(even, cur, 0, ids);
        }
    }
    const Piece done = cur;
    const bool wbad = __any(bad);
    if (more) {
        cur = piece(p_next, b, base);
        ids = ids_next, ahead = ahead_next;
        bad = bad_next;
        load_q(cur);
        if (!ANY) load_tile(even, cur, 0, ids);
    }

    // ---- join the four waves
    l = quad_sum(l);
    if (l16 < rows) {
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < EPC; ++e) {
                    const float x = acc[c * EPC + e][r];
                    if (!again || !(place(c, r)[e] * 0.f == 0.f)) place(c, r)[e] = x;
                }
    }
    if (g == 0) {
        ML[w][l16][0] = m;
        ML[w][l16][1] = wbad ? -1.f : l;
    }
    __syncthreads();
    const int quads = dr / 4;
    for (int u = tid; u < rows * quads; u += kPWaves * 64) {
        const int q = u / quads, d = (u - q * quads) * 4;
        float mt = -INFINITY, lt = 0.f;
        bool rejected = false;
#pragma unroll
        for (int y = 0; y < kPWaves; ++y) mt = fmaxf(mt, ML[y][q][0]);
        const float ms = mt == -INFINITY ? 0.f : mt;
        floatx4 o = floatx4{};
#pragma unroll
        for (int wv = 0; wv < kPWaves; ++wv) {
            const float f = __builtin_amdgcn_exp2f(ML[wv][q][0] - ms), lx = ML[wv][q][1];
            rejected |= lx < 0.f;
            lt = fmaf(lx, f, lt);
            const floatx4 y = *reinterpret_cast<const floatx4 *>(&Os[wv][q][d]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(y[e], f, o[e]);
        }
        if (rejected && u == 0) raise_flag(a.status, CAST_FLAG_BAD_PAGE);
        const int head = done.h * a.G + done.rb * 16 + q;
        if (!done.whole) {
            const int64_t at = (int64_t)(2 * x + (p != p_first)) * a.prows + q;
            *reinterpret_cast<floatx4 *>(a.part_o + at * dr + d) = o;
            if (d == 0) {
                a.part_ml[at * 2] = mt;
                a.part_ml[at * 2 + 1] = rejected ? -1.f : lt;
            }
        } else {
            const float inv = rejected || lt == 0.f ? 0.f : 1.f / (lt * E::kPScale);
            T *op = static_cast<T *>(a.out) + (int64_t)done.b * a.o_req + (int64_t)head * a.o_head + d;
            if (rejected || lt == 0.f) o = floatx4{};
            if constexpr (F32) {
                *reinterpret_cast<floatx4 *>(op) = o * inv;
            } else {
                u32x2 y = {E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
                *reinterpret_cast<u32x2 *>(op) = y;
            }
            if (d == 0 && a.lse)
                a.lse[(int64_t)done.b * a.Hq + head] = rejected || lt == 0.f ? -INFINITY : (ms + log2f(lt)) * kPLn2;
        }
    }
    if (!more) return;
    p = p_next;
    __syncthreads();   // (the join's LDS is read)
    }
}

// Joins the pieces of one (request, query head): groups of LP lanes, one
// float4 of the head dim a lane, walk every NG-th split with up to four in
// flight and their own running maximum, then join through LDS.
template <typename E, int LP>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    using T = typename E::T;
    constexpr int NG = 256 / LP;
    __shared__ __attribute__((aligned(16))) floatx4 Os[NG][LP];
    __shared__ float ML[NG][2];
    const int b = blockIdx.y, head = blockIdx.x;
    const int h = head / a.G, in = head - h * a.G, rb = in / 16, q = in - rb * 16;
    const int32_t *unit = a.units + 2 * (((int64_t)b * a.rbs + rb) * a.Hkv + h);
    const int slot = unit[0], ns = unit[1];
    if (ns <= 1) return;
    // the pieces after the first are their workgroups' first ones
    auto row_of = [&](int s) __attribute__((always_inline)) { return (int64_t)(s ? (slot & ~1) + 2 * s : slot) * a.prows + q; };
    const int grp = threadIdx.x / LP, d = (threadIdx.x % LP) * 4, dl = min(d, a.D - 4);
    float m = -INFINITY, l = 0.f;
    bool rejected = false;
    floatx4 o = floatx4{};
    for (int s0 = grp; s0 < ns; s0 += 4 * NG) {
        floatx4 y[4];
        float mx[4], lx[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t row = row_of(min(s0 + j * NG, ns - 1));
            mx[j] = a.part_ml[row * 2];
            lx[j] = a.part_ml[row * 2 + 1];
            y[j] = *reinterpret_cast<const floatx4 *>(a.part_o + row * a.D + dl);
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            rejected |= lx[j] < 0.f;
            mn = fmaxf(mn, mx[j]);
        }
        const float ms = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        l *= alpha;
        o *= alpha;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (s0 + j * NG >= ns) break;
            const float f = __builtin_amdgcn_exp2f(mx[j] - ms);
            l = fmaf(lx[j], f, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(y[j][e], f, o[e]);
        }
    }
    Os[grp][threadIdx.x % LP] = o;
    if (d == 0) {
        ML[grp][0] = m;
        ML[grp][1] = l;
    }
    rejected = __syncthreads_or(rejected);
    if (grp || d >= a.D) return;
#pragma unroll
    for (int g = 1; g < NG; ++g) m = fmaxf(m, ML[g][0]);
    const float ms = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = floatx4{};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float f = __builtin_amdgcn_exp2f(ML[g][0] - ms);
        l = fmaf(ML[g][1], f, l);
        const floatx4 y = Os[g][threadIdx.x];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(y[e], f, o[e]);
    }
    const bool none = rejected || l == 0.f;
    const float inv = none ? 0.f : 1.f / (l * E::kPScale);
    if (none) o = floatx4{};
    T *op = static_cast<T *>(a.out) + (int64_t)b * a.o_req + (int64_t)head * a.o_head + d;
    if constexpr (E::kBytes == 4) {
        *reinterpret_cast<floatx4 *>(op) = o * inv;
    } else {
        u32x2 y = {E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<u32x2 *>(op) = y;
    }
    if (d == 0 && a.lse) a.lse[(int64_t)b * a.Hq + head] = none ? -INFINITY : (ms + log2f(l)) * kPLn2;
}
template <typename E>
static void launch_join(const PagedAttnArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.Hq, (unsigned)a.batch);
    if (a.D <= 64) paged_join_kernel<E, 16><<<grid, 256, 0, st>>>(a);
    else if (a.D <= 128) paged_join_kernel<E, 32><<<grid, 256, 0, st>>>(a);
    else paged_join_kernel<E, 64><<<grid, 256, 0, st>>>(a);
}

// --------------------------------------------------------------------------
// Host side
// --------------------------------------------------------------------------
struct PagedKernel {
    const void *fn;
    int tile;   // keys of a workgroup's tile
};
template <int D, typename E, bool PAD, bool ANY>
static PagedKernel paged_instance() {
    return {reinterpret_cast<const void *>(&paged_attn_kernel<D, E, PAD, ANY>), 16 * E::kBlocks * kPWaves};
}
// Head dims 64, 128 and 256 have instances of their own; other multiples of 8
// take the next larger one with the rest masked.  Page sizes whose 16-key
// blocks may straddle a page take the instances that look up every key.
template <int D, typename E>
static PagedKernel paged_instance_of(bool pad, bool any) {
    if (any) return paged_instance<D, E, true, true>();
    return pad ? paged_instance<D, E, true, false>() : paged_instance<D, E, false, false>();
}
template <typename E>
static PagedKernel paged_kernel_of(int32_t D, bool any) {
    if (D <= 64) return paged_instance_of<64, E>(D != 64, any);
    if (D <= 128) return paged_instance_of<128, E>(D != 128, any);
    return paged_instance_of<256, E>(D != 256, any);
}
static PagedKernel paged_kernel(int32_t dtype, int32_t D, bool any) {
    if (dtype == CAST_FP32) return paged_kernel_of<PF32>(D, any);
    return dtype == CAST_FP16 ? paged_kernel_of<PFp16>(D, any) : paged_kernel_of<PBf16>(D, any);
}
static bool paged_any(int32_t page_size, int32_t max_pages) { return page_size % 16 != 0 && max_pages > 1; }

// Workgroups of kernel k that the current device holds at once (an MI355X's
// 256 CUs, one each, where no device is visible), looked up once per (device,
// kernel).
struct PagedDevice {
    int slots, cus;
};
static PagedDevice paged_slots(const PagedKernel &k) {
    struct Entry {
        int dev;
        const void *fn;
        PagedDevice d;
    };
    static std::mutex mu;
    static Entry cache[128];
    static int used = 0;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) return {256, 256};
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < used; ++i)
        if (cache[i].dev == dev && cache[i].fn == k.fn) return cache[i].d;
    int n = 0, cus = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, k.fn, kPWaves * 64, 0) != hipSuccess || n < 1) n = 1;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) cus = 256;
    const PagedDevice d{n * cus, cus};
    if (used < 128) cache[used++] = Entry{dev, k.fn, d};
    return d;
}

// Whether units of at most `bytes` of K and V get a workgroup each and no
// pieces, which saves the join's launch (4 to 5 us) and the schedule.  Split
// against whole, us, units of a batch's longest request (or of lengths spread
// evenly below it), 64-key pages, 4 query heads a KV head:
//   bf16, D 128, 256 KB:  32 units 13.2 and 11.0, 256 22.5 and 16.5, 1024 50.2 and 45.4
//   the same, 512 KB:     32 units 13.9 and 16.2, 128 21.4 and 18.4 (17.3 and 17.0), 1024 88.1 and 84.1 (60.1 and 53.1)
//   1 MB:                 128 units 30.9 and 29.3 (26.3 and 27.2), 1024 168 and 165 (98.7 and 98.3)
//   bf16, D 64, 256 KB:   32 units 11.8 and 11.9, 128 15.1 and 12.2, 1024 54.3 and 43.8
//   fp32, D 128, 512 KB:  32 units 13.8 and 19.0, 128 21.3 and 20.5 (18.3 and 19.7), 1024 91.4 and 86.8
//   bf16, D 256, 512 KB:  128 units 24.2 and 22.7 (20.8 and 21.3), 512 54.3 and 52.8, 1024 98.1 and 103.9 (79.2 and 74.1)
// Pages whose keys are looked up one by one (`any`) take a tile twice as long:
//   bf16, D 128, 256 KB:  32 units 13.4 and 15.1, 128 17.2 and 16.1 (16.4 and 15.4), 1024 69.9 and 64.0
//   the same, 512 KB:     128 units 22.6 and 26.4 (19.1 and 25.1)
// 1 MB would pay from 256 units of like lengths on, but there one long request
// among short ones would keep all waiting.
static bool paged_whole(int64_t bytes, int64_t units, bool any, int cus) {
    return (any ? 2 * bytes : bytes) <= (2 * units >= cus ? 512 << 10 : 256 << 10);
}

struct PagedPlan {
    int32_t wgs, least, cut, cus;   // as PagedAttnArgs
    bool fits;            // tile indices fit 31 bits for any lengths
};
static PagedPlan paged_plan(int32_t batch, int32_t max_pages, int32_t page_size, int32_t Hq, int32_t Hkv, int32_t D,
                            int32_t window, int32_t dtype, int32_t kv_split) {
    const bool any = paged_any(page_size, max_pages);
    const PagedKernel k = paged_kernel(dtype, D, any);
    const int64_t units = (int64_t)batch * Hkv * ((Hq / Hkv + 15) / 16);
    int64_t keys = (int64_t)max_pages * page_size;
    if (window > 0 && window < keys) keys = (int64_t)window + k.tile - 1;   // (a window may start inside a tile)
    const int64_t tiles = (keys + k.tile - 1) / k.tile;
    const int64_t least = kv_split > 0 ? ((int64_t)kv_split + k.tile - 1) / k.tile : kMinTiles;
    const PagedDevice d = paged_slots(k);
    const bool whole = kv_split < 0 || tiles <= least ||
                       (kv_split == 0 && paged_whole(tiles * k.tile * D * (dtype == CAST_FP32 ? 8 : 4), units, any, d.cus));
    if (whole) return {units > INT_MAX ? 0 : (int32_t)units, 0, 0, 0, units <= INT_MAX};
    if (units > INT_MAX / (tiles + piece_cost(64))) return {0, 0, 0, 0, false};
    const int64_t most = units * ((tiles + least - 1) / least);
    const int64_t wgs = kv_split > 0 ? most : std::min<int64_t>(most, d.slots);
    return {(int32_t)wgs, (int32_t)least, kv_split > 0, d.cus, true};
}
static size_t p_align256(size_t x) { return (x + 255) & ~(size_t)255; }
struct PagedParts {
    size_t ml, o, all;   // offsets of the partials' sums and outputs, bytes in all
};
static PagedParts paged_parts(const PagedPlan &p, int32_t batch, int32_t Hkv, int32_t G, int32_t D) {
    const size_t rows = (size_t)2 * p.wgs * std::min(G, 16);
    PagedParts s{};
    s.ml = p_align256((size_t)batch * Hkv * ((G + 15) / 16) * 2 * sizeof(int32_t));
    s.o = s.ml + p_align256(rows * 2 * sizeof(float));
    s.all = p.least ? s.o + p_align256(rows * D * sizeof(float)) : 0;
    return s;
}

}  // namespace cast

using namespace cast;

extern "C" size_t cast_paged_attn_workspace_size(int32_t batch, int32_t max_pages, int32_t page_size,
                                                 int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                 int32_t window, int32_t dtype, int32_t kv_split) {
    if (batch <= 0 || max_pages <= 0 || page_size <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
        num_q_heads % num_kv_heads || head_dim <= 0 || head_dim % 8 || head_dim > 256)
        return 0;
    if (dtype != CAST_BF16 && dtype != CAST_FP16 && dtype != CAST_FP32) return 0;
    return paged_parts(paged_plan(batch, max_pages, page_size, num_q_heads, num_kv_heads, head_dim, window, dtype, kv_split),
                       batch, num_kv_heads, num_q_heads / num_kv_heads, head_dim).all;
}

extern "C" int cast_paged_attn_fwd(const void *q, const void *k_pages, const void *v_pages, void *out, float *lse,
                                   const int32_t *page_table, int64_t table_ld, int32_t max_pages, int32_t n_pages,
                                   int32_t page_size, const int32_t *seq_len, int32_t batch, int32_t num_q_heads,
                                   int32_t num_kv_heads, int32_t head_dim, int64_t q_req, int64_t q_head,
                                   int64_t kp_page, int64_t kp_head, int64_t kp_tok, int64_t vp_page, int64_t vp_head,
                                   int64_t vp_tok, int64_t o_req, int64_t o_head, int32_t dtype, float sm_scale,
                                   float softcap, int32_t window, int32_t kv_split, void *workspace,
                                   size_t workspace_bytes, int32_t *status, cast_stream_t stream) {
    if (batch < 0 || max_pages < 0 || n_pages < 0 || page_size <= 0 || window < 0 || head_dim <= 0) return CAST_ERR_SHAPE;
    if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads) return CAST_ERR_HEAD_RATIO;
    if (dtype != CAST_BF16 && dtype != CAST_FP16 && dtype != CAST_FP32) return CAST_ERR_DTYPE;
    if (head_dim % 8 || head_dim > 256) return CAST_ERR_HEAD_DIM;
    if (!(sm_scale > 0.f) || !isfinite(sm_scale) || !(softcap >= 0.f) || !isfinite(softcap)) return CAST_ERR_SCALE;
    if (batch == 0) return CAST_OK;
    // every request's visible keys need a page to be read from
    if (max_pages == 0 || n_pages == 0) return CAST_ERR_SHAPE;
    if ((int64_t)max_pages * page_size > INT32_MAX - 512) return CAST_ERR_SHAPE;
    if (!q || !k_pages || !v_pages || !out || !page_table || !seq_len) return CAST_ERR_NULL_POINTER;
    const int64_t esz = dtype == CAST_FP32 ? 4 : 2;
    auto a16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (!a16(q) || !a16(k_pages) || !a16(v_pages) || !a16(out)) return CAST_ERR_ALIGNMENT;
    const int64_t strides[10] = {q_req, q_head, kp_page, kp_head, kp_tok, vp_page, vp_head, vp_tok, o_req, o_head};
    for (int64_t s : strides)
        if ((s * esz) % 16) return CAST_ERR_ALIGNMENT;
    // a lane's offsets within 16 rows are 32 bits
    if (kp_tok < 0 || vp_tok < 0 || kp_tok * esz >= 1 << 27 || vp_tok * esz >= 1 << 27) return CAST_ERR_SHAPE;
    const bool any = paged_any(page_size, max_pages);
    const PagedPlan p = paged_plan(batch, max_pages, page_size, num_q_heads, num_kv_heads, head_dim, window, dtype, kv_split);
    if (!p.fits || batch > 65535 || num_q_heads > 65535) return CAST_ERR_SHAPE;
    const PagedParts parts = paged_parts(p, batch, num_kv_heads, num_q_heads / num_kv_heads, head_dim);
    if (parts.all) {
        if (!workspace) return CAST_ERR_NULL_POINTER;
        if (workspace_bytes < parts.all) return CAST_ERR_WORKSPACE;
        if (reinterpret_cast<uintptr_t>(workspace) & 255) return CAST_ERR_ALIGNMENT;
    }
    PagedAttnArgs a{};
    a.q = q;
    a.k = k_pages;
    a.v = v_pages;
    a.out = out;
    a.lse = lse;
    a.table = page_table;
    a.seq_len = seq_len;
    a.status = status;
    a.table_ld = table_ld;
    a.q_req = q_req;
    a.q_head = q_head;
    a.o_req = o_req;
    a.o_head = o_head;
    a.kp_page = kp_page * esz;
    a.kp_head = kp_head * esz;
    a.kp_tok = kp_tok * esz;
    a.vp_page = vp_page * esz;
    a.vp_head = vp_head * esz;
    a.vp_tok = vp_tok * esz;
    a.n_pages = n_pages;
    a.page_size = page_size;
    a.by_page = fast_div((uint32_t)page_size);
    a.batch = batch;
    a.Hq = num_q_heads;
    a.Hkv = num_kv_heads;
    a.G = num_q_heads / num_kv_heads;
    a.rbs = (a.G + 15) / 16;
    a.D = head_dim;
    a.cap = max_pages * page_size;
    a.window = window;
    a.wgs = p.wgs;
    a.least = p.least;
    a.cut = p.cut;
    a.cus = p.cus;
    a.prows = std::min(a.G, 16);
    a.softcap = softcap;
    a.scale = softcap > 0.f ? sm_scale : sm_scale * kPLog2e;
    if (parts.all) {
        char *ws = static_cast<char *>(workspace);
        a.units = reinterpret_cast<int32_t *>(ws);
        a.part_ml = reinterpret_cast<float *>(ws + parts.ml);
        a.part_o = reinterpret_cast<float *>(ws + parts.o);
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    void *args[] = {&a};
    const PagedKernel k = paged_kernel(dtype, head_dim, any);
    if (hipLaunchKernel(k.fn, dim3((unsigned)p.wgs), dim3(kPWaves * 64), args, 0, st) != hipSuccess) return CAST_ERR_HIP;
    if (p.least) {
        if (dtype == CAST_FP32) launch_join<PF32>(a, st);
        else if (dtype == CAST_FP16) launch_join<PFp16>(a, st);
        else launch_join<PBf16>(a, st);
        if (hipGetLastError() != hipSuccess) return CAST_ERR_HIP;
    }
    return CAST_OK;
}
