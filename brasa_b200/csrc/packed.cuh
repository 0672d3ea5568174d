// Device-side pieces of the operators over a packed run (several new tokens per sequence, see brasa_packed_run): whose a row is, and where
// a position lies in the pool. Everything read from device tables is held against the buffers' sizes before it becomes an address.
#pragma once
#include "attn_device.cuh"

namespace brasa_dev {

struct PackedView {
    const int32_t *table;   // [seqs][max_pages]
    const uint32_t *lens, *starts;
    uint32_t seqs, max_pages, num_pages, tokens, longest, hkv;
};

// The last sequence that begins at or before row t: the warp looks at 32 boundaries at a time. UINT32_MAX when none does.
__device__ __forceinline__ uint32_t packed_sequence(const uint32_t *starts, uint32_t seqs, uint32_t t, uint32_t lane) {
    uint32_t lo = 0, n = seqs;  // (starts[lo] <= t once a boundary was found)
    bool found = false;
    while (n > 1 || !found) {
        const uint32_t step = (n + 31) / 32, at = lane * step;
        const uint32_t c = __popc(__ballot_sync(0xffffffffu, at < n && starts[lo + at] <= t));
        if (c == 0) return UINT32_MAX;
        found = true;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
    return lo;
}

// Row t of a run: its sequence and position; false for a row that is nobody's (behind the last sequence, past `longest`, starts that fall).
__device__ __forceinline__ bool packed_row(const PackedView &p, uint32_t t, uint32_t lane, uint32_t &seq, uint32_t &pos) {
    seq = packed_sequence(p.starts, p.seqs, t, lane);
    if (seq == UINT32_MAX || t >= p.starts[seq + 1]) return false;
    const uint32_t j = t - p.starts[seq];
    const uint64_t at = (uint64_t)p.lens[seq] + j;
    pos = (uint32_t)min(at, (uint64_t)UINT32_MAX);
    return j < p.longest;
}

// Page of a position, or -1 where there is none.
__device__ __forceinline__ int32_t packed_page(const PackedView &p, uint32_t seq, uint32_t pos) {
    const uint32_t i = pos / BRASA_KV_PAGE;
    if (i >= p.max_pages) return -1;
    const int32_t page = p.table[(size_t)seq * p.max_pages + i];
    return (uint32_t)page < p.num_pages ? page : -1;
}

// two signed bytes of `w` (already without sign bit: +128), chosen by `sel` into the low bytes of two halves, as f16 (exact) times a pair of scales
__device__ __forceinline__ uint32_t bytes_h2(uint32_t w, uint32_t sel, __half2 scale) {
    const uint32_t u = __byte_perm(w, 0x64646464u, sel);  // 1024 + byte
    __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));  // - 1152
    h = __hmul2(h, scale);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// F16 precision forms weights as 2^(s - m + 7): with scores up to m + 8 the largest is 2^15, near f16's end, so that 2^-25, where f16 loses its last bit, is 2^-32 of
// the weight of a score of m. (O and l carry the factor alike; a part's m is given without it.)
constexpr float WEIGHT_LOG2 = 7.0f;
__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < INFINITY); }

// ---- the work of a run in a line, cut evenly ----
// An item is up to item_tokens tokens of one sequence, each with the heads of a key head's group, against that key head. In the line an item takes `start`
// units for its beginning and end and one per 2^tile_log2 keys that its last token sees. Equal pieces of the line go to the blocks; a block works
// through the items of its piece, whole ones and parts. A piece's end that falls within `snap` units of an item's ends moves there, since a
// part costs a way through memory and a merge. Everything is read from device memory, so that a recorded launch follows new lengths.
struct PackedLine {
    PackedView v;
    uint32_t group, inv, item_tokens;        // query heads per key head, 65 536 / group rounded up
    uint32_t tile_log2, start, snap, least;  // ..; fewest units that are worth a block
    uint32_t min_rows, max_rows;             // sequences of fewer or more rows (tokens times group) are another kernel's
};
inline PackedLine packed_line(const PackedView &v, uint32_t group, uint32_t rows_item, uint32_t tile_log2, uint32_t start, uint32_t snap, uint32_t least, uint32_t min_rows, uint32_t max_rows) {
    return PackedLine{v, group, (65536 + group - 1) / group, rows_item / group, tile_log2, start, snap, least, min_rows, max_rows};
}
// token of a row of an item (below 2^10, for groups up to 8)
__device__ __forceinline__ uint32_t row_token(const PackedLine &l, uint32_t r) { return r * l.inv >> 16; }
struct PackedItem {
    uint64_t first;             // its place in the line
    uint32_t seq, t0, n, past;  // sequence, its first row of the run, its tokens, the positions before them
    uint32_t part, kh, tiles;   // which item_tokens of its tokens, key head, key tiles
    uint32_t j;                 // the key tile that a piece begins or ends at
};

__device__ __forceinline__ void line_sequence(const PackedLine &l, uint32_t s, PackedItem &it) {
    const uint32_t a = min(l.v.starts[s], l.v.tokens), b = min(l.v.starts[s + 1], l.v.tokens), past = l.v.lens[s];
    const uint64_t most = (uint64_t)l.v.max_pages * BRASA_KV_PAGE;
    uint64_t n = min(b > a ? b - a : 0u, l.v.longest);
    n = past >= most ? 0 : min(n, most - past);
    const uint64_t rows = n * l.group;
    it.seq = s;
    it.t0 = a;
    it.past = past;
    it.n = rows >= l.min_rows && rows <= l.max_rows ? (uint32_t)n : 0u;
}
__device__ __forceinline__ uint32_t line_keys(const PackedLine &l, const PackedItem &it) { return it.past + min((it.part + 1) * l.item_tokens, it.n); }  // that its last token sees
__device__ __forceinline__ uint32_t line_tokens(const PackedLine &l, const PackedItem &it) { return min(l.item_tokens, it.n - it.part * l.item_tokens); }
__device__ __forceinline__ uint32_t line_tiles(const PackedLine &l, const PackedItem &it) { return ((line_keys(l, it) - 1) >> l.tile_log2) + 1; }
// units of all items of a sequence, for one key head
__device__ __forceinline__ uint64_t line_units(const PackedLine &l, const PackedItem &it) {
    uint64_t u = 0;
#pragma unroll 4
    for (uint32_t t = l.item_tokens; t < it.n; t += l.item_tokens) u += l.start + 1 + ((it.past + t - 1) >> l.tile_log2);
    return it.n ? u + l.start + 1 + ((it.past + it.n - 1) >> l.tile_log2) : 0;
}

// What a block leaves of the items at its piece's ends, for the kernel that adds parts up.
struct PackedNote {
    uint32_t opens;   // the piece began an item and left it open: the rest of the note is about that item
    uint32_t closes;  // the piece ended an item that began before it
    uint32_t t0, rows, kh;  // its first row of the run, its rows (tokens times group), key head
};
// floats of a part's slot: O [rows_item][128], m and l by row
__host__ __device__ constexpr size_t packed_part_floats(uint32_t rows_item) { return (size_t)rows_item * 130; }

struct PackedPieces {
    uint64_t sums[32], total;
    PackedItem at[2];  // where this block's piece begins and ends
    uint32_t pieces;   // how many there are
};
// All threads of the block (a multiple of 32). False when this block has no piece.
template <uint32_t THREADS>
__device__ bool line_cut(const PackedLine &l, PackedPieces &w) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid >= THREADS) {  // (more threads than take part: they only keep the barriers company)
        for (int i = 0; i < 3; ++i) __syncthreads();
        return blockIdx.x < w.pieces;
    }
    const uint32_t each = (l.v.seqs + THREADS - 1) / THREADS, s0 = min(tid * each, l.v.seqs), s1 = min(s0 + each, l.v.seqs);
    PackedItem it;
    uint64_t mine = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        line_sequence(l, s, it);
        mine += line_units(l, it) * l.v.hkv;
    }
    uint64_t upto = mine;
    for (uint32_t x = 1; x < 32; x <<= 1) {
        const uint64_t o = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += o;
    }
    if (lane == 31) w.sums[warp] = upto;
    __syncthreads();
    uint64_t total = 0;
    for (uint32_t i = 0; i < THREADS / 32; ++i) {
        if (i == warp) upto += total;
        total += w.sums[i];
    }
    const uint32_t pieces = (uint32_t)min((uint64_t)gridDim.x, (total + l.least - 1) / l.least);
    if (tid == 0) {
        w.total = total;
        w.pieces = pieces;
        w.at[1].first = total;  // (unless the line goes on there)
        w.at[1].j = 0;
    }
    __syncthreads();
    if (blockIdx.x < pieces) {
        for (uint32_t e = 0; e < 2; ++e) {
            const uint64_t unit = total * (blockIdx.x + e) / pieces;
            if (unit < upto - mine || unit >= upto) continue;
            uint64_t first = upto - mine;
            uint32_t s = s0;
            for (;; ++s) {  // (ends: the unit lies in one of this thread's sequences)
                line_sequence(l, s, it);
                if (each == 1) break;
                const uint64_t u = line_units(l, it) * l.v.hkv;
                if (unit < first + u) break;
                first += u;
            }
            // of the sequence's items, in one key head's units: part by part (their key heads lie behind one another)
            uint64_t left = unit - first;
            uint32_t each_item = 0;
            for (it.part = 0;; ++it.part) {  // (ends: the unit lies in one of them)
                it.tiles = line_tiles(l, it);
                each_item = l.start + it.tiles;
                const uint64_t all = (uint64_t)each_item * l.v.hkv;
                if (left < all) break;
                left -= all;
            }
            it.kh = (uint32_t)(left / each_item);
            const uint32_t tiles = it.tiles;
            it.first = unit - left + (uint64_t)it.kh * each_item;
            const uint32_t off = (uint32_t)(unit - it.first);
            it.j = off > l.start ? off - l.start : 0u;
            if (it.j < l.snap) it.j = 0;
            else if (tiles - it.j < l.snap) it.j = tiles;  // (as far as the item goes: the next piece begins behind it)
            w.at[e] = it;
        }
    }
    __syncthreads();
    return blockIdx.x < pieces;
}
// The item behind `it`; false at the end of the line.
__device__ __forceinline__ bool line_next(const PackedLine &l, PackedItem &it) {
    it.first += l.start + it.tiles;
    it.j = 0;
    if (++it.kh < l.v.hkv) return true;
    it.kh = 0;
    if (++it.part * l.item_tokens >= it.n) {
        it.part = 0;
        do {
            if (++it.seq >= l.v.seqs) return false;
            line_sequence(l, it.seq, it);
        } while (it.n == 0);
    }
    it.tiles = line_tiles(l, it);
    return true;
}

// ---- rows before a value that is not finite ----
// A weight of zero times an infinity or NaN of V is NaN, so that in a matrix product a key behind a row's own position, new in the same run, reaches the row. A kernel
// that finds a row not finite although keys of its share lie behind it comes here with all its threads, at a place where no other warp waits for them.
// V of the share is looked at once, dim by dim: where the first NaN and the first infinity of either sign are, and the last of them. That says of a dim which a value behind
// the row reached what it has to be when the row sees such values itself: NaN, or the infinity. Only where it sees none the row is taken again, key by key. An
// overflowing channel or a prompt of NaN so costs the one look. An 8-bit value that the products round to an f16 infinity is one. Weights in two terms make NaN of an
// infinity that the row does see, since the second term is 0 or negative: such a kernel comes here with every row that is not finite.
template <int KV, bool HALF>
constexpr bool two_terms() { return KV == BRASA_KV_F16 && !HALF; }
struct PackedAgain {
    const float *q;
    const uint8_t *kpool, *vpool;
    void *o;
    float *part;  // the share's slot, when it is not the whole of its item's keys
    uint32_t hq;
    float scale;
    uint32_t seq, kh, t0, rows, past;  // of the item: its first row of the run, its rows, positions before its first token
    uint32_t from, upto, rows_item;    // keys of the share; rows of a slot
    bool whole;
};
struct PackedRowSums {
    float m, l;
    float4 o;
};
template <int KV>
__device__ __forceinline__ float4 packed_row4(const uint8_t *row, uint32_t lane) {
    const float2 a = tile_at2<KV>(row, 4 * lane), b = tile_at2<KV>(row, 4 * lane + 2);
    return make_float4(a.x, a.y, b.x, b.y);
}
// The sums of one row over the keys [from, to), a warp, four dims a lane: m, the sum of 2^(s - m) and that times V. Backwards, until nothing is left that is not NaN.
template <int KV>
__device__ __forceinline__ PackedRowSums packed_row_again(const PackedView &v, const uint8_t *kpool, const uint8_t *vpool, const float *q, float scale, uint32_t seq, uint32_t kh, uint32_t from, uint32_t to) {
    constexpr uint32_t AT_ONCE = 8;  // (half a page)
    const uint32_t lane = threadIdx.x & 31;
    const float4 x = reinterpret_cast<const float4 *>(q)[lane];
    const float c = scale * 1.4426950408889634f;
    PackedRowSums r{-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    for (uint32_t n = to > from ? (to - from + AT_ONCE - 1) / AT_ONCE : 0; n > 0; --n) {  // (from is a multiple of 64)
        const uint32_t k0 = from + (n - 1) * AT_ONCE;
        const int32_t page = packed_page(v, seq, k0);
        if (page < 0) continue;
        float s[AT_ONCE];
        float4 y[AT_ONCE];
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; ++e) {
            const size_t at = (((size_t)page * BRASA_KV_PAGE + (k0 + e) % BRASA_KV_PAGE) * v.hkv + kh) * KvRow<KV>::BYTES;
            y[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            s[e] = -INFINITY;
            if (k0 + e < to) {
                const float4 k = packed_row4<KV>(kpool + at, lane);
                y[e] = packed_row4<KV>(vpool + at, lane);
                s[e] = fmaf(x.w, k.w, fmaf(x.z, k.z, fmaf(x.y, k.y, x.x * k.x)));
                for (int i = 16; i > 0; i >>= 1) s[e] += __shfl_xor_sync(0xffffffffu, s[e], i);
                s[e] *= c;
            }
        }
        float now = r.m;
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; ++e) now = fmaxf(now, s[e]);
        const float ref = now == -INFINITY ? 0.0f : now, f = r.m == -INFINITY ? 0.0f : exp2_approx(r.m - ref);
        r.m = now;
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; ++e) {
            const float w = exp2_approx(s[e] - ref);
            l += w;
            o = make_float4(fmaf(w, y[e].x, o.x), fmaf(w, y[e].y, o.y), fmaf(w, y[e].z, o.z), fmaf(w, y[e].w, o.w));
        }
        r.l = fmaf(r.l, f, l);
        r.o = make_float4(fmaf(r.o.x, f, o.x), fmaf(r.o.y, f, o.y), fmaf(r.o.z, f, o.z), fmaf(r.o.w, f, o.w));
        if (__all_sync(0xffffffffu, r.o.x != r.o.x && r.o.y != r.o.y && r.o.z != r.o.z && r.o.w != r.o.w)) break;
    }
    return r;
}
template <int KV, bool HALF>
__device__ __noinline__ void packed_rows_again(const PackedLine &l, const PackedAgain &a) {
    __shared__ uint32_t first_nan[128], first_up[128], first_down[128], past_bad[128];  // by dim: positions, the last one further on
    constexpr float LIMIT = KV == BRASA_KV_Q8_0 && HALF ? 65520.0f : INFINITY;
    constexpr bool TERMS = two_terms<KV, HALF>();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (uint32_t i = threadIdx.x; i < 128; i += blockDim.x) {
        first_nan[i] = first_up[i] = first_down[i] = UINT32_MAX;
        past_bad[i] = 0;
    }
    __syncthreads();
#pragma unroll 4
    for (uint32_t p = a.from + warp; p < a.upto; p += warps) {
        const int32_t page = packed_page(l.v, a.seq, p);
        if (page < 0) continue;
        const float4 y = packed_row4<KV>(a.vpool + (((size_t)page * BRASA_KV_PAGE + p % BRASA_KV_PAGE) * l.v.hkv + a.kh) * KvRow<KV>::BYTES, lane);
        const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (!(fabsf(ys[e]) < LIMIT)) {
                atomicMax(&past_bad[4 * lane + e], p + 1);
                atomicMin(&(ys[e] != ys[e] ? first_nan : ys[e] > 0.0f ? first_up : first_down)[4 * lane + e], p);
            }
    }
    __syncthreads();
    for (uint32_t r = warp; r < a.rows; r += warps) {
        const uint32_t token = row_token(l, r), own = a.past + token;
        const size_t at = ((size_t)(a.t0 + token) * a.hq + a.kh * l.group + r - token * l.group) * 128 + 4 * lane;
        auto put = [&](const float4 &v) {
            if (!a.whole) reinterpret_cast<float4 *>(a.part + (size_t)r * 128)[lane] = v;
            else if (HALF) {
                const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
                *reinterpret_cast<uint2 *>(static_cast<__half *>(a.o) + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
            } else *reinterpret_cast<float4 *>(static_cast<float *>(a.o) + at) = v;
        };
        float4 y;
        if (!a.whole) y = reinterpret_cast<const float4 *>(a.part + (size_t)r * 128)[lane];
        else if (HALF) {
            const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const __half *>(a.o) + at);
            const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
            y = make_float4(lo.x, lo.y, hi.x, hi.y);
        } else y = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.o) + at);
        float ys[4] = {y.x, y.y, y.z, y.w};
        bool clean = false, dead = false, known = false, taken = false;  // a dim without such values; one that is NaN, so that a score is; a dim known to be an infinity; one not known
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t d = 4 * lane + e, bad = past_bad[d];
            if (bad == 0) {
                clean = true;
                dead = dead || ys[e] != ys[e];
            } else if (not_finite(ys[e]) && (TERMS || bad > own + 1) && first_nan[d] > own) {
                const bool up = first_up[d] <= own, down = first_down[d] <= own;
                if (up != down) {
                    ys[e] = up ? INFINITY : -INFINITY;
                    known = true;
                } else if (!up) taken = true;
            }
        }
        if (__any_sync(0xffffffffu, dead)) continue;
        const bool some = __any_sync(0xffffffffu, known);
        if (!__any_sync(0xffffffffu, taken) && (!some || __any_sync(0xffffffffu, clean))) {  // (with no dim clean a NaN of a score would not show)
            if (some) put(make_float4(ys[0], ys[1], ys[2], ys[3]));
            continue;
        }
        const PackedRowSums x = packed_row_again<KV>(l.v, a.kpool, a.vpool, a.q + at - 4 * lane, a.scale, a.seq, a.kh, a.from, min(a.upto, own + 1));
        const float inv = !a.whole ? 1.0f : x.l == 0.0f ? 0.0f : 1.0f / x.l;
        put(make_float4(x.o.x * inv, x.o.y * inv, x.o.z * inv, x.o.w * inv));
        if (!a.whole && lane == 0) {
            a.part[(size_t)a.rows_item * 128 + r] = x.m;
            a.part[(size_t)a.rows_item * 129 + r] = x.l;
        }
    }
    __syncthreads();
}

}  // namespace brasa_dev
