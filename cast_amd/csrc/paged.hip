// K6: new tokens' K and V into a cache of pages, rotated to their positions
// on the way.
//
// The reference keeps its per-request store in place (cast_trees/serving.py:
// 191-205, appended to by _append_store, 264-289, as K4 does here) and leaves
// the rotation to the model.  Here the cache is a pool of pages that a table
// hands out per request: token slot t of request b lies in page
// table[b][t / page_size] at offset t % page_size, and row j of a request's
// new tokens goes to slot seq_len[b] + j.  With cos / sin tables, element
// pairs (x, y) of the first rot_dim elements of every K (and Q) head become
//   (x cos - y sin, y cos + x sin)
// of the token's position, computed in float and rounded once to the cache's
// type (products of 16-bit elements with 24-bit angles have no shorter exact
// form).  Pairs are (i, i + rot/2), or adjacent elements.
//
// Memory-bound: every row is read once and written once in 16-byte chunks.
// One thread moves one chunk (one pair of chunks where the two halves of a
// head rotate into each other); a workgroup's threads belong to one token (or
// two), so its slot is looked up once, by scalar loads.  Measured: six prompts of
// up to 4k tokens (8 KV and 32 query heads of 128, bf16) 359 MB in 71 us a call,
// 5.05 TB/s, a copy's rate; a token each of 8 requests 3.4 us.
#include "cast_common.hpp"

namespace cast {

constexpr int kPagedLayersPerLaunch = 64;   // four base addresses each in the kernel arguments (2 KiB)
constexpr int kPagedThreads = 256;
constexpr int kPathRows = 8;                // workgroups that share a request's accepted rows
// Rows of a workgroup: two once a row each gives more workgroups than the device
// holds (8 a CU), so that a second round becomes a second load in flight.  One
// against two: 512 rows (32 + 8 heads of 128, bf16, 1024 workgroups) 6.3 and 6.8
// us, 1024 rows 9.5 and 9.3, 4096 26.4 and 25.1; prompts of 13k rows 79 and 71
// (four: 71 to 72); fp32, 256 rows 6.2 and 6.5, 512 8.8 and 8.6, 4096 45.6 and 42.3.
constexpr int64_t kOneRowGroups = 2048;

struct PagedAppendArgs {
    const void *q;
    void *q_out, *k_out;
    const float *cos, *sin;
    const int32_t *table, *seq_len, *cu_q, *path, *path_len, *positions;
    int32_t *new_len, *status;
    int64_t table_ld, rope_ld;
    int64_t k_tok, k_head, v_tok, v_head, kp_page, kp_head, kp_tok, vp_page, vp_head, vp_tok;   // bytes
    int64_t q_tok, q_head, qo_tok, qo_head, ko_tok, ko_head;                                    // bytes
    int32_t max_pages, n_pages, page_size, batch, total, path_stride, max_pos;
    int32_t Hq, Hkv;        // Hq = 0: no q
    int32_t chunks;         // 16-byte chunks per head
    int32_t rot_chunks;     // of which the first ones rotate
    int32_t interleaved;
    int32_t units;          // threads per rotated head: a pair of chunks each in the half style
    int32_t tasks;          // threads per token
    int32_t rows;           // rows to move (path: kPathRows workgroups a request); the workgroups (x) behind theirs check one request each
};

// The layers' addresses of one launch, of 1 or kPagedLayersPerLaunch layers:
// a launch copies its arguments, and 2 KiB of them show in a small call.
template <int LAYERS>
struct PagedLayers {
    const void *k[LAYERS], *v[LAYERS];
    void *k_pages[LAYERS], *v_pages[LAYERS];
};

// Row j of request b: source row, slot, page and offset, and the rotation's
// table row; ok when all of them lie inside their tables.
struct PagedRow {
    int32_t src, page, offset, pos;
    int32_t flags;   // why not (cast_device_flag)
};

__device__ __forceinline__ PagedRow paged_row(const PagedAppendArgs &a, int b, int root, int j, int S) {
    PagedRow r{root + j, 0, 0, 0, 0};
    if (a.path && j > 0) {
        const int node = a.path[(int64_t)b * a.path_stride + j - 1];
        if (node < 0 || node >= a.total) {
            r.flags = CAST_FLAG_BAD_OFFSETS;
            return r;
        }
        r.src = root + node + 1;
    }
    const int64_t slot = (int64_t)S + j;
    if (S < 0 || r.src < 0 || r.src >= a.total || slot >= (int64_t)a.max_pages * a.page_size) {
        r.flags = CAST_FLAG_BAD_OFFSETS;
        return r;
    }
    const uint32_t at = (uint32_t)slot / (uint32_t)a.page_size;
    r.page = a.table[(int64_t)b * a.table_ld + at];
    r.offset = (int32_t)((uint32_t)slot - at * (uint32_t)a.page_size);
    if (r.page < 0 || r.page >= a.n_pages) r.flags |= CAST_FLAG_BAD_PAGE;
    if (a.cos) {
        r.pos = a.positions ? a.positions[r.src] : (int32_t)slot;
        if (r.pos < 0 || r.pos >= a.max_pos) r.flags |= CAST_FLAG_BAD_POSITION;
    }
    return r;
}

// Request b's first row and row count (no row where they make no sense).
__device__ __forceinline__ bool paged_request(const PagedAppendArgs &a, int b, int &root, int &n) {
    if (a.path) {
        root = a.cu_q[b];
        n = a.path_len[b] + 1;
        return root >= 0 && root < a.total && n >= 1 && n <= kMaxPack;
    }
    root = a.cu_q ? a.cu_q[b] : b;
    n = a.cu_q ? a.cu_q[b + 1] - root : 1;
    return root >= 0 && n >= 0 && (int64_t)root + n <= a.total;
}

// The request of packed row `row` - as many as end at or before it - with its
// first row, end and length in the cache: one round of loads per 64 requests.
__device__ __forceinline__ int request_of(const PagedAppendArgs &a, int row, int &root, int &end, int &S) {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = min(b0 + lane, a.batch - 1);
        const int c0 = a.cu_q[b], c1 = a.cu_q[b + 1], len = a.seq_len[b];
        const uint64_t past = __ballot(c1 <= row);
        if (~past) {
            const int at = __builtin_ctzll(~past);
            root = __builtin_amdgcn_readlane(c0, at);
            end = __builtin_amdgcn_readlane(c1, at);
            S = __builtin_amdgcn_readlane(len, at);
            return b0 + at;
        }
    }
    return a.batch;
}

// One chunk's elements as floats, and back.
template <typename E>
__device__ __forceinline__ void widen_chunk(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bits = w[i];
        x[2 * i] = E::widen((uint16_t)bits);
        x[2 * i + 1] = E::widen((uint16_t)(bits >> 16));
    }
}
// (A float is made of every rotated element first: fp16 has an instruction that
// rounds a fused product straight to 16 bits, and the compiler takes it in one
// instance and not in another, where a row should have the same bits in a call
// of any size.)
template <typename E>
__device__ __forceinline__ u32x4 round_chunk(float (&x)[8]) {
    if constexpr (__is_same(E, Fp16)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("" : "+v"(x[i]));
    }
    return u32x4{E::pack2(x[0], x[1]), E::pack2(x[2], x[3]), E::pack2(x[4], x[5]), E::pack2(x[6], x[7])};
}
struct Fp32 {};
template <>
__device__ __forceinline__ void widen_chunk<Fp32>(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bits = w[i];   // (a bit cast of the element itself reads element 0)
        x[i] = __builtin_bit_cast(float, bits);
    }
}
template <>
__device__ __forceinline__ u32x4 round_chunk<Fp32>(float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, x[i]);
    return w;
}

template <int N>
__device__ __forceinline__ void load_angles(const float *p, float (&x)[8]) {
    if constexpr (N == 2) {
        x[0] = p[0];
        x[1] = p[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const floatx4 w = *reinterpret_cast<const floatx4 *>(p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i + j] = w[j];
        }
    }
}

template <typename E, int LAYERS, int ROWS>
__global__ __launch_bounds__(kPagedThreads) void paged_append_kernel(PagedAppendArgs a, PagedLayers<LAYERS> at) {
    constexpr int EPC = __is_same(E, Fp32) ? 4 : 8;   // elements per 16-byte chunk
    const int layer = LAYERS == 1 ? 0 : blockIdx.z;
    const int groups = ROWS == 1 ? a.rows : (int)(((uint32_t)a.rows + ROWS - 1) / ROWS);   // workgroups that move rows
    if ((int)blockIdx.x >= groups) {
        // ---- one request's check, by its own workgroup: any row that cannot
        // be placed leaves its length as it was
        if (blockIdx.y || layer) return;
        const int b = blockIdx.x - groups;
        const int S = a.seq_len[b];
        int root, n;
        int32_t flags = 0;
        // (where offsets decrease, rows may have gone to another request)
        if (a.cu_q && !a.path)
            for (int i = threadIdx.x; i < a.batch; i += kPagedThreads) flags |= a.cu_q[i + 1] < a.cu_q[i] ? CAST_FLAG_BAD_OFFSETS : 0;
        if (!paged_request(a, b, root, n)) {
            flags = CAST_FLAG_BAD_OFFSETS;
        } else {
            for (int j = threadIdx.x; j < n; j += kPagedThreads) flags |= paged_row(a, b, root, j, S).flags;
        }
        if (flags) raise_flag(a.status, flags);
        const int bad = __syncthreads_or(flags);
        if (threadIdx.x == 0 && a.new_len) a.new_len[b] = bad ? S : S + n;
        return;
    }
    // ---- this thread's chunk: q heads, then k heads, then v heads
    const int task = blockIdx.y * kPagedThreads + threadIdx.x;
    const bool live = task < a.tasks;
    int head = 0, unit = 0, kind = 2;   // 0: q, 1: k, 2: v
    const int turned = (a.Hq + a.Hkv) * a.units;
    if (task < turned) {
        head = (int)((uint32_t)task / (uint32_t)a.units);
        unit = task - head * a.units;
        kind = head < a.Hq ? 0 : 1;
        if (kind) head -= a.Hq;
    } else {
        const int t = task - turned;
        head = (int)((uint32_t)t / (uint32_t)a.chunks);
        unit = t - head * a.chunks;
    }
    // half style: units [0, rot_chunks / 2) hold chunk pairs, the others one chunk
    const int half = a.rot_chunks >> 1;
    const bool paired = kind < 2 && !a.interleaved && unit < half;
    const int chunk = kind < 2 && !a.interleaved && !paired ? unit + half : unit;

    const int64_t far = half * 16;   // from a pair's first chunk to its second
    const char *rows = static_cast<const char *>(kind == 0 ? a.q : kind == 1 ? at.k[layer] : at.v[layer]);
    const int64_t row_step = kind == 0 ? a.q_tok : kind == 1 ? a.k_tok : a.v_tok;
    rows += head * (kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head) + chunk * 16;
    auto load = [&](int64_t src, u32x4 &x, u32x4 &y) __attribute__((always_inline)) {
        if (!live) return;
        x = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(rows + src * row_step));   // (read once: 83.5 -> 80 us for 13k tokens)
        if (paired) y = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(rows + src * row_step + far));
    };
    auto put = [&](const PagedRow &r, u32x4 x, u32x4 y) __attribute__((always_inline)) {
        char *to, *also = nullptr;   // also: k_out
        const int64_t src = r.src;
        if (kind == 0) {
            to = static_cast<char *>(a.q_out) + src * a.qo_tok + head * a.qo_head;
        } else if (kind == 1) {
            to = static_cast<char *>(at.k_pages[layer]) + r.page * a.kp_page + head * a.kp_head + r.offset * a.kp_tok;
            if (a.k_out) also = static_cast<char *>(a.k_out) + src * a.ko_tok + head * a.ko_head + chunk * 16;
        } else {
            to = static_cast<char *>(at.v_pages[layer]) + r.page * a.vp_page + head * a.vp_head + r.offset * a.vp_tok;
        }
        to += chunk * 16;
        if (paired) {
            float xf[8], yf[8], c[8], s[8], xr[8], yr[8];
            load_angles<EPC>(a.cos + r.pos * a.rope_ld + chunk * EPC, c);
            load_angles<EPC>(a.sin + r.pos * a.rope_ld + chunk * EPC, s);
            widen_chunk<E>(x, xf);
            widen_chunk<E>(y, yf);
#pragma unroll
            for (int i = 0; i < EPC; ++i) {
                xr[i] = fmaf(xf[i], c[i], -(yf[i] * s[i]));
                yr[i] = fmaf(yf[i], c[i], xf[i] * s[i]);
            }
            x = round_chunk<E>(xr);
            y = round_chunk<E>(yr);
            *reinterpret_cast<u32x4 *>(to + far) = y;
            if (also) *reinterpret_cast<u32x4 *>(also + far) = y;
        } else if (kind < 2 && a.interleaved && chunk < a.rot_chunks) {
            float xf[8], c[8], s[8], xr[8];
            load_angles<EPC / 2>(a.cos + r.pos * a.rope_ld + chunk * (EPC / 2), c);
            load_angles<EPC / 2>(a.sin + r.pos * a.rope_ld + chunk * (EPC / 2), s);
            widen_chunk<E>(x, xf);
#pragma unroll
            for (int i = 0; i < EPC / 2; ++i) {
                xr[2 * i] = fmaf(xf[2 * i], c[i], -(xf[2 * i + 1] * s[i]));
                xr[2 * i + 1] = fmaf(xf[2 * i + 1], c[i], xf[2 * i] * s[i]);
            }
            x = round_chunk<E>(xr);
        }
        *reinterpret_cast<u32x4 *>(to) = x;
        if (also) *reinterpret_cast<u32x4 *>(also) = x;
    };

    if (a.path) {
        const int b = blockIdx.x / kPathRows;
        int root, n;
        if (!paged_request(a, b, root, n)) return;
        const int S = a.seq_len[b];
        for (int j = blockIdx.x % kPathRows; j < n; j += kPathRows) {
            const PagedRow r = paged_row(a, b, root, j, S);
            if (r.flags || !live) continue;
            u32x4 x{}, y{};
            load(r.src, x, y);
            put(r, x, y);
        }
        return;
    }
    // the rows are known: their loads run beside the lookups of where they go
    const int first = blockIdx.x * ROWS;
    u32x4 x[ROWS], y[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (i == 0 || first + i < a.rows) load(first + i, x[i], y[i]);
    PagedRow r[ROWS];
    int b = 0, root = 0, end = first, S = 0;   // the request of rows [root, end)
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = first + i;
        r[i].flags = CAST_FLAG_BAD_OFFSETS;
        if (i && row >= a.rows) continue;
        if (!a.cu_q) {
            b = root = row;
            S = a.seq_len[b];
        } else if (row >= end) {
            b = request_of(a, row, root, end, S);
            // rows behind the last request, offsets that make no sense
            if (b >= a.batch || root < 0 || root > row || end > a.total) {
                end = row;
                continue;
            }
        }
        r[i] = paged_row(a, b, root, row - root, S);
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (!r[i].flags) put(r[i], x[i], y[i]);
}

template <int LAYERS, int ROWS>
static int launch_append(const PagedAppendArgs &a, const void *const *k, const void *const *v, void *const *k_pages,
                         void *const *v_pages, int32_t n, int32_t dtype, dim3 grid, hipStream_t st) {
    PagedLayers<LAYERS> at{};
    for (int32_t l = 0; l < n; ++l) {
        at.k[l] = k[l];
        at.v[l] = v[l];
        at.k_pages[l] = k_pages[l];
        at.v_pages[l] = v_pages[l];
    }
    if (dtype == CAST_BF16) paged_append_kernel<Bf16, LAYERS, ROWS><<<grid, kPagedThreads, 0, st>>>(a, at);
    else if (dtype == CAST_FP16) paged_append_kernel<Fp16, LAYERS, ROWS><<<grid, kPagedThreads, 0, st>>>(a, at);
    else paged_append_kernel<Fp32, LAYERS, ROWS><<<grid, kPagedThreads, 0, st>>>(a, at);
    return hipGetLastError() == hipSuccess ? CAST_OK : CAST_ERR_HIP;
}

}  // namespace cast

using namespace cast;

extern "C" int cast_paged_append(const void *const *k, const void *const *v, void *const *k_pages,
                                 void *const *v_pages, int32_t layers, const int32_t *page_table, int64_t table_ld,
                                 int32_t max_pages, int32_t n_pages, int32_t page_size, const int32_t *seq_len,
                                 int32_t *new_len, int32_t batch, int32_t total, const int32_t *cu_q,
                                 const int32_t *path, int32_t path_stride, const int32_t *path_len, const void *q,
                                 void *q_out, void *k_out, const float *cos, const float *sin, int64_t rope_ld,
                                 int32_t max_pos, int32_t rot_dim, int32_t interleaved, const int32_t *positions,
                                 int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t k_tok,
                                 int64_t k_head, int64_t v_tok, int64_t v_head, int64_t kp_page, int64_t kp_head,
                                 int64_t kp_tok, int64_t vp_page, int64_t vp_head, int64_t vp_tok, int64_t q_tok,
                                 int64_t q_head, int64_t qo_tok, int64_t qo_head, int64_t ko_tok, int64_t ko_head,
                                 int32_t dtype, int32_t *status, cast_stream_t stream) {
    if (layers < 0 || batch < 0 || total < 0 || max_pages < 0 || n_pages < 0 || page_size <= 0 || num_kv_heads <= 0 ||
        head_dim <= 0)
        return CAST_ERR_SHAPE;
    if (dtype != CAST_BF16 && dtype != CAST_FP16 && dtype != CAST_FP32) return CAST_ERR_DTYPE;
    if (layers == 0 || batch == 0) return CAST_OK;
    if (!k || !v || !k_pages || !v_pages || !seq_len || (max_pages && !page_table)) return CAST_ERR_NULL_POINTER;
    if (path && (!path_len || !cu_q)) return CAST_ERR_NULL_POINTER;
    if (path && path_stride < kMaxPack) return CAST_ERR_SHAPE;
    if (!cu_q && batch > total) return CAST_ERR_SHAPE;
    if ((int64_t)max_pages * page_size > INT32_MAX) return CAST_ERR_SHAPE;
    const int64_t esz = dtype == CAST_FP32 ? 4 : 2, epc = 16 / esz;
    if (head_dim % epc || head_dim * esz > 16 * 1024) return CAST_ERR_HEAD_DIM;
    // q, k_out and the rotation belong to one layer's forward; accepted rows
    // (path) were rotated by it
    const bool rope = cos != nullptr || sin != nullptr;
    if ((rope || q || k_out) && (layers != 1 || path)) return CAST_ERR_SHAPE;
    if ((q != nullptr) != (q_out != nullptr) || (cos != nullptr) != (sin != nullptr)) return CAST_ERR_NULL_POINTER;
    if (q && (num_q_heads <= 0 || num_q_heads % num_kv_heads)) return CAST_ERR_HEAD_RATIO;
    if (rope && (rot_dim <= 0 || rot_dim > head_dim || rot_dim % (2 * epc))) return CAST_ERR_HEAD_DIM;
    if (rope && (max_pos < 0 || rope_ld < rot_dim / 2)) return CAST_ERR_SHAPE;
    auto a16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if (rope && (!a16(cos) || !a16(sin) || rope_ld % 4)) return CAST_ERR_ALIGNMENT;
    if (!a16(q) || !a16(q_out) || !a16(k_out)) return CAST_ERR_ALIGNMENT;
    const int64_t strides[16] = {k_tok,  k_head, v_tok, v_head, kp_page, kp_head, kp_tok,  vp_page,
                                 vp_head, vp_tok, q_tok, q_head, qo_tok,  qo_head, ko_tok, ko_head};
    for (int i = 0; i < 16; ++i)
        if ((i < 10 || (i < 14 ? q != nullptr : k_out != nullptr)) && (strides[i] * esz) % 16) return CAST_ERR_ALIGNMENT;
    for (int32_t l = 0; l < layers; ++l) {
        if (!k[l] || !v[l] || !k_pages[l] || !v_pages[l]) return CAST_ERR_NULL_POINTER;
        if (!a16(k[l]) || !a16(v[l]) || !a16(k_pages[l]) || !a16(v_pages[l])) return CAST_ERR_ALIGNMENT;
    }
    // new_len is written while other workgroups (and later launches) still
    // read these
    if (new_len) {
        auto overlaps = [&](const int32_t *p, int64_t n) {
            const uintptr_t a0 = reinterpret_cast<uintptr_t>(new_len), a1 = a0 + (uintptr_t)batch * 4;
            const uintptr_t b0 = reinterpret_cast<uintptr_t>(p), b1 = b0 + (uintptr_t)n * 4;
            return p && a0 < b1 && b0 < a1;
        };
        if (overlaps(seq_len, batch) || overlaps(cu_q, (int64_t)batch + 1) || overlaps(path_len, batch) ||
            overlaps(path, (int64_t)batch * path_stride) || overlaps(positions, total) ||
            overlaps(page_table, (batch - 1) * table_ld + max_pages))
            return CAST_ERR_ALIAS;
    }
    PagedAppendArgs a{};
    a.q = q;
    a.q_out = q_out;
    a.k_out = k_out;
    a.cos = cos;
    a.sin = sin;
    a.table = page_table;
    a.seq_len = seq_len;
    a.cu_q = cu_q;
    a.path = path;
    a.path_len = path_len;
    a.positions = positions;
    a.status = status;
    a.table_ld = table_ld;
    a.rope_ld = rope_ld;
    int64_t *const bytes[16] = {&a.k_tok,   &a.k_head, &a.v_tok, &a.v_head, &a.kp_page, &a.kp_head, &a.kp_tok, &a.vp_page,
                                &a.vp_head, &a.vp_tok, &a.q_tok, &a.q_head, &a.qo_tok,  &a.qo_head, &a.ko_tok, &a.ko_head};
    for (int i = 0; i < 16; ++i) *bytes[i] = strides[i] * esz;
    a.max_pages = max_pages;
    a.n_pages = n_pages;
    a.page_size = page_size;
    a.batch = batch;
    a.total = total;
    a.path_stride = path_stride;
    a.max_pos = max_pos;
    a.Hq = q ? num_q_heads : 0;
    a.Hkv = num_kv_heads;
    a.chunks = (int32_t)(head_dim / epc);
    a.rot_chunks = rope ? (int32_t)(rot_dim / epc) : 0;
    a.interleaved = interleaved != 0;
    a.units = a.interleaved ? a.chunks : a.chunks - a.rot_chunks / 2;
    const int64_t tasks = (int64_t)(a.Hq + a.Hkv) * a.units + (int64_t)a.Hkv * a.chunks;
    const int64_t slices = (tasks + kPagedThreads - 1) / kPagedThreads;
    if (slices > 65535) return CAST_ERR_SHAPE;
    a.tasks = (int32_t)tasks;
    const int64_t rows = path ? (int64_t)batch * kPathRows : cu_q ? total : batch;
    if (rows + batch > INT32_MAX) return CAST_ERR_SHAPE;
    a.rows = (int32_t)rows;
    for (int32_t l0 = 0; l0 < layers; l0 += kPagedLayersPerLaunch) {
        const int32_t n = layers - l0 < kPagedLayersPerLaunch ? layers - l0 : kPagedLayersPerLaunch;
        const bool checks = l0 == 0 && (new_len || status);
        a.new_len = checks ? new_len : nullptr;
        const bool two = n == 1 && !path && rows * slices >= kOneRowGroups;
        const dim3 grid((unsigned)((two ? (rows + 1) / 2 : rows) + (checks ? batch : 0)), (unsigned)slices, (unsigned)n);
        if (grid.x == 0) continue;
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        auto *const run = n > 1 ? launch_append<kPagedLayersPerLaunch, 1> : two ? launch_append<1, 2> : launch_append<1, 1>;
        const int rc = run(a, k + l0, v + l0, k_pages + l0, v_pages + l0, n, dtype, grid, st);
        if (rc != CAST_OK) return rc;
    }
    return CAST_OK;
}
