// Norm, RoPE and store, and attention, of a packed run: any number of new tokens per sequence over the paged pool.
#include <math.h>

#include "packed_tc.h"

using namespace brasa_dev;

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE;
constexpr int D = 128;

// y = x / sqrt(mean x^2 + eps) * w of rows of q and k, rotated by the token's own position (pairs i, i + 64), and the store of k and v. Bound by memory: q read
// and written, k and v read, the cache's rows written. A warp takes four rows of a token (a lane four dims of each, so that a row is one
// request and a pair's other half lies sixteen lanes on), asks for all of them first and finds the token's sequence, position and page meanwhile. 9 prompts of
// 7257 tokens (32 heads on 8, f16) 71 us, 4.6 TB/s (one row a warp: 92 us).
constexpr uint32_t STORE_ROWS = 4;

// four dims a lane of one row, rounded to the cache type
template <int KV>
__device__ __forceinline__ void put_row4(uint8_t *row, const float4 &y, uint32_t lane) {
    if (KV == BRASA_KV_F32) reinterpret_cast<float4 *>(row)[lane] = y;
    else if (KV == BRASA_KV_F16) {
        const __half2 a = __floats2half2_rn(y.x, y.y), b = __floats2half2_rn(y.z, y.w);
        reinterpret_cast<uint2 *>(row)[lane] = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {  // blocks of 32 dims, eight lanes each: the largest magnitude / 127 as f16, codes against that
        float top = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
        for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const __half dh = __float2half_rn(__fdiv_rn(top, 127.0f));
        const float d = __half2float(dh);
        auto code = [&](float v) { return (uint32_t)(uint8_t)(int8_t)(d == 0.0f ? 0.0f : fminf(fmaxf(rintf(__fdiv_rn(v, d)), -127.0f), 127.0f)); };
        reinterpret_cast<uint32_t *>(row)[lane] = code(y.x) | code(y.y) << 8 | code(y.z) << 16 | code(y.w) << 24;
        if (lane % 8 == 0) reinterpret_cast<__half *>(row + 128)[lane / 8] = dh;
    }
}

template <int KV>
__global__ void __launch_bounds__(256) qk_norm_rope_store_packed_kernel(const float *q, const float *k, const float *v, const float *q_norm, const float *k_norm,
                                                                        const float *cos_t, const float *sin_t, uint8_t *kpool, uint8_t *vpool, PackedView p,
                                                                        float *q_out, uint32_t hq, float eps, uint32_t per_tok, uint64_t warps) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched as a programmatic dependent: see brasa_launch_dependent)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint64_t w = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31, hkv = p.hkv, rows = hq + 2 * hkv;
    if (w >= warps) return;
    const uint32_t t = (uint32_t)(w / per_tok), r0 = (uint32_t)(w % per_tok) * STORE_ROWS;
    float4 x[STORE_ROWS];
#pragma unroll
    for (uint32_t e = 0; e < STORE_ROWS; ++e) {
        const uint32_t r = min(r0 + e, rows - 1);
        const float *src = r < hq ? q + ((size_t)t * hq + r) * D : (r < hq + hkv ? k + ((size_t)t * hkv + r - hq) * D : v + ((size_t)t * hkv + r - hq - hkv) * D);
        x[e] = reinterpret_cast<const float4 *>(src)[lane];
    }
    uint32_t seq, pos;
    if (!packed_row(p, t, lane, seq, pos) || pos / PAGE >= p.max_pages) return;
    const int32_t page = packed_page(p, seq, pos);
    const size_t slot = (size_t)max(page, 0) * PAGE + pos % PAGE;
    const float4 c = reinterpret_cast<const float4 *>(cos_t + (size_t)pos * (D / 2))[lane & 15], s = reinterpret_cast<const float4 *>(sin_t + (size_t)pos * (D / 2))[lane & 15];
    const float sign = lane < 16 ? -1.0f : 1.0f;
#pragma unroll
    for (uint32_t e = 0; e < STORE_ROWS; ++e) {
        const uint32_t r = r0 + e;
        if (r >= rows) break;
        if (r >= hq + hkv) {
            if (page >= 0) put_row4<KV>(vpool + (slot * hkv + r - hq - hkv) * KvRow<KV>::BYTES, x[e], lane);
            continue;
        }
        float ss = (x[e].x * x[e].x + x[e].y * x[e].y) + (x[e].z * x[e].z + x[e].w * x[e].w);
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float f = 1.0f / sqrtf(ss / (float)D + eps);
        const float4 n = reinterpret_cast<const float4 *>(r < hq ? q_norm : k_norm)[lane];
        float4 y = make_float4(x[e].x * f * n.x, x[e].y * f * n.y, x[e].z * f * n.z, x[e].w * f * n.w), o;
        o.x = __shfl_xor_sync(0xffffffffu, y.x, 16);  // (the pair's other half)
        o.y = __shfl_xor_sync(0xffffffffu, y.y, 16);
        o.z = __shfl_xor_sync(0xffffffffu, y.z, 16);
        o.w = __shfl_xor_sync(0xffffffffu, y.w, 16);
        y = make_float4(y.x * c.x + sign * o.x * s.x, y.y * c.y + sign * o.y * s.y, y.z * c.z + sign * o.z * s.z, y.w * c.w + sign * o.w * s.w);
        if (r < hq) reinterpret_cast<float4 *>(q_out + ((size_t)t * hq + r) * D)[lane] = y;
        else if (page >= 0) put_row4<KV>(kpool + (slot * hkv + r - hq) * KvRow<KV>::BYTES, y, lane);
    }
}

// ---- few rows against many keys: the cache's bytes are the work ------------------------------------------------------------------
// Four warps, 64 keys at a time through a ring of cp.async stages. An item's up to 64 rows are one to four tiles of 16 for mma.sync m16n8k16;
// with one tile the warps share the keys (a page each), with two they go in pairs, with more every warp has a tile of its own. Each warp keeps a
// running maximum, sum and output (the maximum moves only when a score passes it by 2^8), the warps meet at the item's end. The 16 keys of a
// warp's step are one page: a page that is none is skipped, and rows of the cache that the sequence has not reached are never loaded.
// HALF: one f16 term of q * scale and of P, 8-bit rows as f16(d * code): what the F16 precision says. Otherwise q and P enter as two terms, hi + lo, and an f16
// cache's rows as they are. f16 ends at 2^-25, so that both are brought up first, by powers of two: q to a row's largest of 2^14 to 2^15, the weights of a row's 16
// keys to at most 2^15. Hi + lo is then off by 2^-22 of the value, or 2^-40 of the largest, whatever the other keys weigh; a step's product is added to O in 32 bits.
// l sums the weights as the product reads them, by a column of ones beside V.
// Bound by the cache's bytes while an item has one row tile or two, by mma.sync and its waits beyond that, where the tcgen05 kernel takes over (PACKED_TC_MIN_ROWS). 64
// sequences of two to five tokens behind 2600 (32 heads on 8, f16) 154 us, 4.6 TB/s, in F32 precision 198 us; behind a flush of the L2, 16 of three behind 3000 take 61 us with
// an 8-bit cache and 63 with an f16 one: there no unit is full (DRAM 33 %, issue slots 43 %), a page's chain of reads, conversions and products is what is waited for.
struct FewParams {
    PackedLine l;
    const float *q;
    const uint8_t *kpool, *vpool;
    void *o;
    float *part;
    PackedNote *notes;
    uint32_t hq;
    float scale;
    uint32_t late_wait;
};
// FEW_BLOCKS: of an SM. 8 bit, the 16 sequences above and 28 of 2000 to 6000 positions (64 heads on 8): two blocks of four stages 77 and 158 us, three
// of three 81 and 163, four of two 100 and 199 (before the copies had a page to a warp).
constexpr uint32_t FEW_ROWS = 64, FEW_KEYS = 64, FEW_BLOCKS = 2;
template <int KV> struct FewStage;
template <> struct FewStage<BRASA_KV_F16> { static constexpr uint32_t K_PITCH = 256, V_PITCH = 256, STAGES = 3; };
// (pitches at which neither the 8-byte reads of K nor the transposed reads of V meet in a bank)
template <> struct FewStage<BRASA_KV_Q8_0> { static constexpr uint32_t K_PITCH = 160, V_PITCH = 144, STAGES = 4; };
template <int KV> constexpr uint32_t few_stage_bytes() { return FEW_KEYS * (FewStage<KV>::K_PITCH + FewStage<KV>::V_PITCH); }
constexpr uint32_t FEW_TS = D + 4;

__device__ __forceinline__ void cp_zfill16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_zfill8(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(valid ? 8u : 0u) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma_f16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// x, y -> f16 pair and, with two terms, the pair of what its rounding dropped
template <bool HALF>
__device__ __forceinline__ void terms_h2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    if (!HALF) {
        const float2 back = __half22float2(h);
        lo = pack_h2(x - back.x, y - back.y);
    }
}
template <int KV, bool HALF>
__global__ void __launch_bounds__(128, FEW_BLOCKS) attn_packed_few_kernel(const __grid_constant__ FewParams p) {
    // Launched as a programmatic dependent. late_wait: the kernel before this one is the same call's tensor-core form, which has itself waited for what both read
    // and whose output this one does not touch: the two run side by side, and this one waits for the other at its end, so that whoever waits for it has
    // waited for both.
    if (!p.late_wait) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using S = FewStage<KV>;
    constexpr bool Q8 = KV == BRASA_KV_Q8_0;
    static_assert(!Q8 || HALF, "8-bit rows are rounded to f16 here");
    constexpr uint32_t STAGE = few_stage_bytes<KV>(), V_AT = FEW_KEYS * S::K_PITCH, ROW = KvRow<KV>::BYTES;
    constexpr float LOG2E = 1.4426950408889634f, SLACK = 8.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PackedPieces pieces;
    __shared__ float sums[4][2][16];
    __shared__ uint32_t again;  // a row is not finite and may have to be otherwise (packed_rows_again)
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem), hkv = p.l.v.hkv, G = p.l.group;
    PackedNote note{};
    if (!line_cut<128>(p.l, pieces)) {
        if (tid == 0) p.notes[blockIdx.x] = note;
        if (p.late_wait) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    PackedItem it = pieces.at[0];
    const uint64_t end_first = pieces.at[1].first;
    const uint32_t end_j = pieces.at[1].j;
    if (it.j == it.tiles) line_next(p.l, it);
    while (it.first < end_first || (it.first == end_first && it.j < end_j)) {
        const uint32_t j0 = it.j, j1 = it.first == end_first ? end_j : it.tiles;
        const uint32_t token0 = it.part * p.l.item_tokens, t0 = it.t0 + token0, rows = line_tokens(p.l, it) * G, nkeys = line_keys(p.l, it);
        const uint32_t share = rows <= 16 ? 4 : (rows <= 32 ? 2 : 1), kp = warp % share, rt = warp / share;
        const bool active = rt * 16 < rows;
        // ---- copies of 64 keys, a page to a warp and two rows at a time: pages looked up one chunk ahead, what the item's last row does not see as zeros ----
        const int32_t *table = p.l.v.table + (size_t)it.seq * p.l.v.max_pages;
        const size_t page_bytes = (size_t)PAGE * hkv * ROW;
        const uint32_t r2 = lane >> 4, pc = lane & 15, step = 2 * hkv * ROW;
        const uint32_t own = (r2 * hkv + it.kh) * ROW + (Q8 ? 8 : 16) * pc;                                    // this lane's piece of the page's first rows
        const uint32_t tail = ((tid & 15) * hkv + it.kh) * ROW + 128, tail_at = (tid & 63) * (tid < 64 ? S::K_PITCH : S::V_PITCH) + 128 + (tid < 64 ? 0 : V_AT);  // (8 bit: scales)
        int32_t pg[4];
        uint32_t there = 0;  // which pages of the last chunks are, four bits each, the newest lowest
        auto look = [&](uint32_t j) {
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x) {
                const int32_t page = j < j1 && 64 * j + 16 * x < nkeys ? table[4 * j + x] : -1;
                pg[x] = (uint32_t)page < p.l.v.num_pages ? page : -1;
            }
        };
        auto fetch = [&](uint32_t j) {
            uint32_t bits = 0;
            if (j < j1) {
                const uint32_t stage = ring + (j % S::STAGES) * STAGE;
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) bits |= (pg[x] >= 0 ? 1u : 0u) << x;
                const int32_t page = warp & 2 ? (warp & 1 ? pg[3] : pg[2]) : (warp & 1 ? pg[1] : pg[0]);
                const uint32_t first = 64 * j + 16 * warp, left = page >= 0 && first < nkeys ? nkeys - first : 0u;  // rows of the page that are seen (16 or more: all)
                const size_t at = (size_t)max(page, 0) * page_bytes + own;
                const uint8_t *ks = p.kpool + at, *vs = p.vpool + at;
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    const uint32_t row = 16 * warp + 2 * u + r2;
                    const bool ok = 2 * u + r2 < left;
                    if (Q8) {
                        cp_zfill8(stage + row * S::K_PITCH + 8 * pc, ks, ok);
                        cp_zfill8(stage + V_AT + row * S::V_PITCH + 8 * pc, vs, ok);
                    } else {
                        const uint32_t to = stage + row * 256 + ((pc ^ (row & 7)) << 4);
                        cp_zfill16(to, ks, ok);
                        cp_zfill16(to + V_AT, vs, ok);
                    }
                    ks += ok ? step : 0;  // (a pointer stays inside the page)
                    vs += ok ? step : 0;
                }
                if (Q8) {
                    const uint32_t x = (tid & 63) >> 4;
                    const int32_t mine = x & 2 ? (x & 1 ? pg[3] : pg[2]) : (x & 1 ? pg[1] : pg[0]);
                    cp_zfill8(stage + tail_at, (tid < 64 ? p.kpool : p.vpool) + (size_t)max(mine, 0) * page_bytes + tail, mine >= 0 && 64 * j + (tid & 63) < nkeys);
                }
                look(j + 1);
            }
            there = there << 4 | bits;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        look(j0);
#pragma unroll
        for (uint32_t i = 0; i + 1 < S::STAGES; ++i) fetch(j0 + i);
        // ---- q fragments: k-step ks holds dims 16 ks + 2 tq, +1 and + 8 (8-bit rows: 32 (ks / 2) + 8 tq + 4 (ks % 2) .. + 3, so that a lane's codes lie together) ----
        uint32_t qh[8][4], ql[8][4];
        uint32_t seen[2];
        float c[2] = {HALF ? LOG2E : p.scale * LOG2E, HALF ? LOG2E : p.scale * LOG2E};
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t r = rt * 16 + g + 8 * h;
            const bool live = active && r < rows;
            const uint32_t token = live ? row_token(p.l, r) : 0, head = live ? r - token * G : 0;
            seen[h] = live ? it.past + token0 + token + 1 : 0;
            const float *src = p.q + ((size_t)(t0 + token) * p.hq + it.kh * G + head) * D;
            float2 a[8][2];
            float top = 0.0f;
#pragma unroll
            for (uint32_t ks = 0; ks < 8; ++ks) {
                a[ks][0] = a[ks][1] = make_float2(0.0f, 0.0f);
                const uint32_t d0 = Q8 ? 32 * (ks >> 1) + 8 * tq + 4 * (ks & 1) : 16 * ks + 2 * tq, d1 = Q8 ? d0 + 2 : d0 + 8;
                if (live) {
                    a[ks][0] = *reinterpret_cast<const float2 *>(src + d0);
                    a[ks][1] = *reinterpret_cast<const float2 *>(src + d1);
                }
                if (!HALF) top = fmaxf(fmaxf(top, fmaxf(fabsf(a[ks][0].x), fabsf(a[ks][0].y))), fmaxf(fabsf(a[ks][1].x), fabsf(a[ks][1].y)));
            }
            float f = p.scale;
            if (!HALF) {  // the row's largest to [2^14, 2^15), as far as powers of two reach; an infinity stays one
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int at = (int)(__float_as_uint(top) >> 23), up = at == 255 ? 0 : min(14 - (at - 127), 100);
                f = __uint_as_float((uint32_t)(127 + up) << 23);
                c[h] *= __uint_as_float((uint32_t)(127 - up) << 23);
            }
#pragma unroll
            for (uint32_t ks = 0; ks < 8; ++ks) {
                terms_h2<HALF>(a[ks][0].x * f, a[ks][0].y * f, qh[ks][h], ql[ks][h]);
                terms_h2<HALF>(a[ks][1].x * f, a[ks][1].y * f, qh[ks][h + 2], ql[ks][h + 2]);
            }
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(seen[0], seen[1]));  // keys that any row of the tile sees
        float m[2] = {-INFINITY, -INFINITY}, l[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[16][4];  // (l: a column of ones beside V, so that it sums the very P; two of the four are the same sums again)
#pragma unroll
        for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        for (uint32_t j = j0; j < j1; ++j) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
            __syncthreads();  // the chunk is there for all, and the one before it is done with
            const uint32_t bits = there >> (4 * (S::STAGES - 2)) & 15;
            fetch(j + S::STAGES - 1);
            const uint32_t kt = ring + (j % S::STAGES) * STAGE, vt = kt + V_AT;
            for (uint32_t u = kp; u < 4; u += share) {
                const uint32_t key0 = 64 * j + 16 * u;
                if (key0 >= most || !(bits >> u & 1)) continue;
                // ---- S = Q K^T of 16 keys: c[t] rows g (0, 1) and g + 8 (2, 3), keys 8 t + 2 tq, + 1 ----
                float s[2][4];
#pragma unroll
                for (uint32_t t = 0; t < 2; ++t) {
                    s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
                    if (!Q8) {
                        const uint32_t row = 16 * u + 8 * t + (lane & 7);
                        float low[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of the second terms: 0 or of either sign, so that an infinite key's score is what the first ones make it
#pragma unroll
                        for (uint32_t ks = 0; ks < 8; ks += 2) {
                            uint32_t b[4];
                            ldsm_x4(b, kt + row * 256 + (((2 * ks + (lane >> 3)) ^ (row & 7)) << 4));
                            mma_f16(s[t], qh[ks], b[0], b[1]);
                            if (!HALF) mma_f16(low, ql[ks], b[0], b[1]);
                            mma_f16(s[t], qh[ks + 1], b[2], b[3]);
                            if (!HALF) mma_f16(low, ql[ks + 1], b[2], b[3]);
                        }
                        if (!HALF)
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) s[t][e] += not_finite(s[t][e]) ? 0.0f : low[e];
                    } else {
                        const uint8_t *row = smem + (kt - ring) + (16 * u + 8 * t + g) * S::K_PITCH;
                        const uint2 sc = *reinterpret_cast<const uint2 *>(row + 128);
#pragma unroll
                        for (uint32_t b = 0; b < 4; ++b) {
                            const uint2 w = *reinterpret_cast<const uint2 *>(row + 32 * b + 8 * tq);
                            const uint32_t pair = b & 2 ? sc.y : sc.x, d2 = __byte_perm(pair, 0, b & 1 ? 0x3232 : 0x1010);
                            const __half2 d = *reinterpret_cast<const __half2 *>(&d2);
                            const uint32_t w0 = w.x ^ 0x80808080u, w1 = w.y ^ 0x80808080u;
                            mma_f16(s[t], qh[2 * b], bytes_h2(w0, 0x4140, d), bytes_h2(w0, 0x4342, d));
                            mma_f16(s[t], qh[2 * b + 1], bytes_h2(w1, 0x4140, d), bytes_h2(w1, 0x4342, d));
                        }
                    }
                }
                // ---- P = 2^(s - m), in two terms 2^(s - the step's largest + 15): O takes the step's product times what the two differ by ----
                uint32_t ph[4], pl[4];
                bool moved = false;
                float back[2] = {1.0f, 1.0f}, share_of[2] = {1.0f, 1.0f};
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    float x[4], top = -INFINITY;
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t key = key0 + 8 * (e >> 1) + 2 * tq + (e & 1);
                        x[e] = key < seen[h] ? s[e >> 1][2 * h + (e & 1)] * c[h] : -INFINITY;
                        top = fmaxf(top, x[e]);
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (top > m[h] + SLACK || (m[h] == -INFINITY && top > -INFINITY)) {
                        moved = true;
                        back[h] = m[h] == -INFINITY ? 0.0f : exp2_approx(m[h] - top);
                        m[h] = top;
                    }
                    float ref = m[h] == -INFINITY ? 0.0f : m[h] - (HALF ? WEIGHT_LOG2 : 0.0f);
                    if (!HALF) {
                        share_of[h] = exp2_approx(top - ref - 15.0f);
                        ref = top == -INFINITY ? 0.0f : top - 15.0f;
                    }
                    float e[4];
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) e[k] = exp2_approx(x[k] - ref);
                    terms_h2<HALF>(e[0], e[1], ph[h], pl[h]);
                    terms_h2<HALF>(e[2], e[3], ph[h + 2], pl[h + 2]);
                }
                if (__any_sync(0xffffffffu, moved)) {
                    l[0] *= back[0];
                    l[2] *= back[1];
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        o[n][0] *= back[0];
                        o[n][1] *= back[0];
                        o[n][2] *= back[1];
                        o[n][3] *= back[1];
                    }
                }
                // ---- O += P V ----
                const uint32_t vrow = 16 * u + (lane & 15), ones = 0x3C003C00u;
                auto add = [&](float to[4], uint32_t b0, uint32_t b1) {
                    if (HALF) return mma_f16(to, ph, b0, b1);
                    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_f16(x, pl, b0, b1);
                    mma_f16(x, ph, b0, b1);
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) to[k] = fmaf(x[k], share_of[k >> 1], to[k]);
                };
                add(l, ones, ones);
                if (!Q8) {
#pragma unroll
                    for (uint32_t n = 0; n < 16; n += 2) {
                        uint32_t b[4];
                        ldsm_x4_t(b, vt + vrow * 256 + (((n + (lane >> 4)) ^ (vrow & 7)) << 4));
                        add(o[n], b[0], b[1]);
                        add(o[n + 1], b[2], b[3]);
                    }
                } else {  // (a transposed 16-bit read brings two dims of two keys: n-tile 2 x holds dims 16 x + 2 col, 2 x + 1 those + 1)
                    uint2 sc[4];  // scales of keys 2 tq, 2 tq + 1, and + 8
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        sc[k] = *reinterpret_cast<const uint2 *>(smem + (vt - ring) + (16 * u + 2 * tq + (k & 1) + 8 * (k >> 1)) * S::V_PITCH + 128);
#pragma unroll
                    for (uint32_t x = 0; x < 8; x += 2) {
                        uint32_t b[4];
                        ldsm_x4_t(b, vt + vrow * S::V_PITCH + 16 * (x + (lane >> 4)));
                        const uint32_t sel = x & 2 ? 0x7632 : 0x5410;
                        const uint32_t d0 = x < 4 ? __byte_perm(sc[0].x, sc[1].x, sel) : __byte_perm(sc[0].y, sc[1].y, sel);
                        const uint32_t d1 = x < 4 ? __byte_perm(sc[2].x, sc[3].x, sel) : __byte_perm(sc[2].y, sc[3].y, sel);
                        const __half2 e0 = *reinterpret_cast<const __half2 *>(&d0), e1 = *reinterpret_cast<const __half2 *>(&d1);
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) {
                            const uint32_t w0 = b[2 * k] ^ 0x80808080u, w1 = b[2 * k + 1] ^ 0x80808080u;
                            mma_f16(o[2 * (x + k)], ph, bytes_h2(w0, 0x4240, e0), bytes_h2(w1, 0x4240, e1));
                            mma_f16(o[2 * (x + k) + 1], ph, bytes_h2(w0, 0x4341, e0), bytes_h2(w1, 0x4341, e1));
                        }
                    }
                }
            }
        }
        // ---- the warps meet: their outputs over the ring ----
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        float *os = reinterpret_cast<float *>(smem) + warp * 16 * FEW_TS;
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            if (tq == 0) {
                sums[warp][0][g + 8 * h] = m[h] - (HALF ? WEIGHT_LOG2 : 0.0f);
                sums[warp][1][g + 8 * h] = l[2 * h];
            }
#pragma unroll
            for (uint32_t n = 0; n < 16; ++n) {
                float *to = os + (g + 8 * h) * FEW_TS;
                if (!Q8) *reinterpret_cast<float2 *>(to + 8 * n + 2 * tq) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                else {
                    to[16 * (n >> 1) + 4 * tq + (n & 1)] = o[n][2 * h];
                    to[16 * (n >> 1) + 4 * tq + 2 + (n & 1)] = o[n][2 * h + 1];
                }
            }
        }
        if (tid == 0) again = 0;
        __syncthreads();
        const bool whole = j0 == 0 && j1 == it.tiles;
        const uint32_t upto = min(nkeys, 64 * j1);
        float *part = p.part + (size_t)(2 * blockIdx.x + (j0 == 0)) * packed_part_floats(FEW_ROWS);
        for (uint32_t r = 0; r < rows; ++r) {
            const uint32_t w0 = r / 16 * share, x = r % 16;
            float M = -INFINITY, L = 0.0f, acc = 0.0f;
            for (uint32_t w = w0; w < w0 + share; ++w) M = fmaxf(M, sums[w][0][x]);
            for (uint32_t w = w0; w < w0 + share; ++w) {
                const float f = sums[w][0][x] == -INFINITY ? 0.0f : exp2_approx(sums[w][0][x] - M);
                L = fmaf(sums[w][1][x], f, L);
                acc = fmaf(reinterpret_cast<float *>(smem)[(w * 16 + x) * FEW_TS + tid], f, acc);
            }
            if (not_finite(acc) && (!HALF || it.past + token0 + row_token(p.l, r) + 1 < upto)) again = 1;
            if (whole) {
                const uint32_t token = row_token(p.l, r);
                const size_t at = ((size_t)(t0 + token) * p.hq + it.kh * G + r - token * G) * D + tid;
                const float v = L == 0.0f ? 0.0f : acc / L;
                if (HALF) static_cast<__half *>(p.o)[at] = __float2half_rn(v);
                else static_cast<float *>(p.o)[at] = v;
            } else {
                part[r * D + tid] = acc;
                if (tid == 0) {
                    part[FEW_ROWS * D + r] = M;
                    part[FEW_ROWS * D + FEW_ROWS + r] = L;
                }
            }
        }
        if (!whole && j0 == 0) note = PackedNote{1, note.closes, t0, rows, it.kh};
        if (j0 > 0 && j1 == it.tiles) note.closes = 1;
        __syncthreads();  // the ring and the sums are free again
        if (again) packed_rows_again<KV, HALF>(p.l, PackedAgain{p.q, p.kpool, p.vpool, p.o, part, p.hq, p.scale, it.seq, it.kh, t0, rows, it.past + token0, 64 * j0, upto, FEW_ROWS, whole});
        if (j1 < it.tiles || !line_next(p.l, it)) break;
    }
    if (tid == 0) p.notes[blockIdx.x] = note;
    if (p.late_wait) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- 32-bit arithmetic: an f32 cache, or an 8-bit one whose values keep all their bits -------------------------------------------------------------
// A block has up to 64 rows and takes 64 keys at a time as f32 in shared memory, K's next tile on its way while V's is used. 256 threads in a square: scores four
// rows by four keys each (keys 16 apart, so that a quarter warp's reads of K meet in no bank), outputs four rows by eight dims. Bound by the FMA units
// with many rows, by the cache's bytes with few: 2100 prompt tokens (8 heads on 2) 331 us, 27 TFLOP/s, 64 sequences of two to five tokens behind 2600 (32 on 8) 826 us, 1.7 TB/s
// (each behind a flush of the L2).
constexpr uint32_t F32_THREADS = 256, F32_P = 68;
constexpr size_t F32_SMEM = (3 * 64 * (size_t)FEW_TS + 64 * F32_P) * sizeof(float);

template <int KV, bool HALF>
__global__ void __launch_bounds__(F32_THREADS, 1) attn_packed_f32_kernel(const __grid_constant__ FewParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) float fs[];
    __shared__ PackedPieces pieces;
    __shared__ uint32_t again;  // a row is not finite and may have to be otherwise (packed_rows_again)
    float *qs = fs, *ks = qs + 64 * FEW_TS, *vs = ks + 64 * FEW_TS, *ps = vs + 64 * FEW_TS;
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, hkv = p.l.v.hkv, G = p.l.group;
    PackedNote note{};
    if (!line_cut<F32_THREADS>(p.l, pieces)) {
        if (tid == 0) p.notes[blockIdx.x] = note;
        return;
    }
    PackedItem it = pieces.at[0];
    const uint64_t end_first = pieces.at[1].first;
    const uint32_t end_j = pieces.at[1].j;
    if (it.j == it.tiles) line_next(p.l, it);
    const float c = p.scale * 1.4426950408889634f;
    while (it.first < end_first || (it.first == end_first && it.j < end_j)) {
        const uint32_t j0 = it.j, j1 = it.first == end_first ? end_j : it.tiles, token0 = it.part * p.l.item_tokens, t0 = it.t0 + token0, rows = line_tokens(p.l, it) * G, nkeys = line_keys(p.l, it);
        const int32_t *table = p.l.v.table + (size_t)it.seq * p.l.v.max_pages;
        auto page_at = [&](uint32_t key) {  // of a position, -1 where there is none or nothing is seen
            const int32_t page = key < nkeys ? table[key / PAGE] : -1;
            return (uint32_t)page < p.l.v.num_pages ? page : -1;
        };
        auto fetch = [&](float *to, const uint8_t *pool, uint32_t j) {  // 64 rows, what is not there as zeros
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint32_t i = tid + F32_THREADS * u, row = i >> 5, pc = i & 31, key = 64 * j + row;
                const int32_t page = j < j1 ? page_at(key) : -1;
                const uint8_t *src = pool + (((size_t)max(page, 0) * PAGE + (key & 15)) * hkv + it.kh) * KvRow<KV>::BYTES;
                if (KV == BRASA_KV_F32) cp_zfill16((uint32_t)__cvta_generic_to_shared(to + row * FEW_TS + 4 * pc), src + 16 * pc, page >= 0);
                else {
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (page >= 0) {
                        const char4 q = reinterpret_cast<const char4 *>(src)[pc];
                        const float d = __half2float(reinterpret_cast<const __half *>(src + 128)[pc >> 3]);
                        v = make_float4(d * (float)q.x, d * (float)q.y, d * (float)q.z, d * (float)q.w);
                    }
                    *reinterpret_cast<float4 *>(to + row * FEW_TS + 4 * pc) = v;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        fetch(ks, p.kpool, j0);
        for (uint32_t i = tid; i < 64 * 32; i += F32_THREADS) {
            const uint32_t r = i >> 5, token = row_token(p.l, r);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < rows) v = reinterpret_cast<const float4 *>(p.q + ((size_t)(t0 + token) * p.hq + it.kh * G + r - token * G) * D)[i & 31];
            *reinterpret_cast<float4 *>(qs + r * FEW_TS + 4 * (i & 31)) = v;
        }
        float m[4], l[4], o[4][8];
        uint32_t seen[4];
#pragma unroll
        for (uint32_t a = 0; a < 4; ++a) {
            const uint32_t r = 4 * ty + a;
            seen[a] = r < rows ? it.past + token0 + row_token(p.l, r) + 1 : 0;
            m[a] = -INFINITY;
            l[a] = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) o[a][e] = 0.0f;
        }
        const bool live = 4 * ty < rows;
        for (uint32_t j = j0; j < j1; ++j) {
            fetch(vs, p.vpool, j);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();  // K and q are there
            float s[4][4];
#pragma unroll
            for (uint32_t a = 0; a < 4; ++a)
#pragma unroll
                for (uint32_t b = 0; b < 4; ++b) s[a][b] = 0.0f;
            if (live) {
#pragma unroll 4
                for (uint32_t d = 0; d < D; d += 4) {
                    float4 x[4], y[4];
#pragma unroll
                    for (uint32_t a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4 *>(qs + (4 * ty + a) * FEW_TS + d);
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) y[b] = *reinterpret_cast<const float4 *>(ks + (tx + 16 * b) * FEW_TS + d);
#pragma unroll
                    for (uint32_t a = 0; a < 4; ++a)
#pragma unroll
                        for (uint32_t b = 0; b < 4; ++b)
                            s[a][b] = fmaf(x[a].w, y[b].w, fmaf(x[a].z, y[b].z, fmaf(x[a].y, y[b].y, fmaf(x[a].x, y[b].x, s[a][b]))));
                }
                bool there[4];
#pragma unroll
                for (uint32_t b = 0; b < 4; ++b) there[b] = page_at(64 * j + 16 * b) >= 0;  // (a thread's keys lie a page apart)
#pragma unroll
                for (uint32_t a = 0; a < 4; ++a) {
                    float top = -INFINITY;
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) {
                        s[a][b] = there[b] && 64 * j + tx + 16 * b < seen[a] ? s[a][b] * c : -INFINITY;
                        top = fmaxf(top, s[a][b]);
                    }
                    for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffu << (tid & 16), top, x));
                    const float now = fmaxf(m[a], top), ref = now == -INFINITY ? 0.0f : now, f = m[a] == -INFINITY ? 0.0f : exp2_approx(m[a] - ref);
                    m[a] = now;
                    float sum = 0.0f;
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) {
                        const float w = exp2_approx(s[a][b] - ref);
                        sum += w;
                        ps[(4 * ty + a) * F32_P + tx + 16 * b] = w;
                    }
                    l[a] = fmaf(l[a], f, sum);
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) o[a][e] *= f;
                }
            }
            __syncthreads();  // K is done with
            fetch(ks, p.kpool, j + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();  // V is there
            if (live) {
                float t[4][8];  // of this tile alone: one key that outweighs all others would swallow theirs one by one
#pragma unroll
                for (uint32_t a = 0; a < 4; ++a)
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) t[a][e] = 0.0f;
#pragma unroll 2
                for (uint32_t k = 0; k < 64; k += 4) {
                    float4 w[4];
#pragma unroll
                    for (uint32_t a = 0; a < 4; ++a) w[a] = *reinterpret_cast<const float4 *>(ps + (4 * ty + a) * F32_P + k);
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const float4 y0 = *reinterpret_cast<const float4 *>(vs + (k + e) * FEW_TS + 4 * tx), y1 = *reinterpret_cast<const float4 *>(vs + (k + e) * FEW_TS + 64 + 4 * tx);
#pragma unroll
                        for (uint32_t a = 0; a < 4; ++a) {
                            const float f = e == 0 ? w[a].x : (e == 1 ? w[a].y : (e == 2 ? w[a].z : w[a].w));
                            t[a][0] = fmaf(f, y0.x, t[a][0]);
                            t[a][1] = fmaf(f, y0.y, t[a][1]);
                            t[a][2] = fmaf(f, y0.z, t[a][2]);
                            t[a][3] = fmaf(f, y0.w, t[a][3]);
                            t[a][4] = fmaf(f, y1.x, t[a][4]);
                            t[a][5] = fmaf(f, y1.y, t[a][5]);
                            t[a][6] = fmaf(f, y1.z, t[a][6]);
                            t[a][7] = fmaf(f, y1.w, t[a][7]);
                        }
                    }
                }
#pragma unroll
                for (uint32_t a = 0; a < 4; ++a)
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) o[a][e] += t[a][e];
            }
            __syncthreads();  // V and the weights are done with
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (tid == 0) again = 0;
        __syncthreads();
        const bool whole = j0 == 0 && j1 == it.tiles;
        const uint32_t upto = min(nkeys, 64 * j1);
        float *part = p.part + (size_t)(2 * blockIdx.x + (j0 == 0)) * packed_part_floats(FEW_ROWS);
        if (live) {
#pragma unroll
            for (uint32_t a = 0; a < 4; ++a) {
                const uint32_t r = 4 * ty + a;
                for (int x = 8; x > 0; x >>= 1) l[a] += __shfl_xor_sync(0xffffu << (tid & 16), l[a], x);
                if (r >= rows) continue;
                bool bad = false;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) bad = bad || not_finite(o[a][e]);
                if (bad && seen[a] < upto) again = 1;
                if (whole) {
                    const uint32_t token = row_token(p.l, r);
                    const size_t at = ((size_t)(t0 + token) * p.hq + it.kh * G + r - token * G) * D + 4 * tx;
                    const float inv = l[a] == 0.0f ? 0.0f : 1.0f / l[a];
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        const float4 v = make_float4(o[a][4 * e] * inv, o[a][4 * e + 1] * inv, o[a][4 * e + 2] * inv, o[a][4 * e + 3] * inv);
                        if (HALF) *reinterpret_cast<uint2 *>(static_cast<__half *>(p.o) + at + 64 * e) = make_uint2(pack_h2(v.x, v.y), pack_h2(v.z, v.w));
                        else *reinterpret_cast<float4 *>(static_cast<float *>(p.o) + at + 64 * e) = v;
                    }
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e)
                        *reinterpret_cast<float4 *>(part + r * D + 64 * e + 4 * tx) = make_float4(o[a][4 * e], o[a][4 * e + 1], o[a][4 * e + 2], o[a][4 * e + 3]);
                    if (tx == 0) {
                        part[FEW_ROWS * D + r] = m[a];
                        part[FEW_ROWS * D + FEW_ROWS + r] = l[a];
                    }
                }
            }
        }
        if (!whole && j0 == 0) note = PackedNote{1, note.closes, t0, rows, it.kh};
        if (j0 > 0 && j1 == it.tiles) note.closes = 1;
        __syncthreads();  // (q's place is free)
        if (again) packed_rows_again<KV, HALF>(p.l, PackedAgain{p.q, p.kpool, p.vpool, p.o, part, p.hq, p.scale, it.seq, it.kh, t0, rows, it.past + token0, 64 * j0, upto, FEW_ROWS, whole});
        if (j1 < it.tiles || !line_next(p.l, it)) break;
    }
    if (tid == 0) p.notes[blockIdx.x] = note;
}

// What either kernel left of the items that several blocks worked on.
struct PackedParts {
    const float *part;
    const PackedNote *notes;
    uint32_t pieces, rows_item, spread;  // blocks, rows of an item, merging blocks to a piece
};
// Such an item is the work of the piece that began and left it open, each of that piece's `spread` blocks with every spread * 8-th row: the sum of 2^(m - M) O over
// that of 2^(m - M) l, O in the order of the keys, l in that of a tree: the same every time. Latency bounds it, so that notes, weights and parts are asked for many at a time.
template <bool HALF>
__global__ void __launch_bounds__(256) attn_packed_merge_kernel(PackedParts a, PackedParts b, void *o, uint32_t hq, PackedLine l) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const bool first = blockIdx.x < a.pieces * a.spread;
    const PackedParts &p = first ? a : b;
    const uint32_t at = first ? blockIdx.x : blockIdx.x - a.pieces * a.spread, piece = at / p.spread, share = at % p.spread, rows_item = p.rows_item;
    const float *part = p.part;
    const PackedNote *notes = p.notes, n = notes[piece];
    if (!n.opens || piece + 1 == p.pieces) return;  // (the line ends with a whole item)
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t step = packed_part_floats(rows_item);
    uint32_t last = piece + 1;  // the piece that ends the item: mostly the next, otherwise 32 of them looked at together
    if (last + 1 < p.pieces && !notes[last].closes)
        for (uint32_t bits = 0; !bits;) {
            const uint32_t k = last + 1 + lane;
            bits = __ballot_sync(0xffffffffu, k + 1 >= p.pieces || notes[k].closes);
            last += bits ? __ffs(bits) : 32;
        }
    for (uint32_t r = share * 8 + warp; r < n.rows; r += p.spread * 8) {
        const float *ms = part + rows_item * D + r, *ls = ms + rows_item, *os = part + (size_t)r * D + 4 * lane;
        // (slot 2 b + 1 is what piece b left open, slot 2 k piece k's share of an item that began before it)
        auto slot = [&](uint32_t k) { return (k == piece ? 2 * (size_t)k + 1 : 2 * (size_t)k) * step; };
        float M = -INFINITY;
        for (uint32_t k = piece + lane; k <= last; k += 32) M = fmaxf(M, ms[slot(k)]);
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        float L = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // Few parts: everything of a part asked for at once. Many (one row over many pieces): a part's weight to a lane, then only the parts themselves (one token behind
        // 16 000: 64 -> 46 us; with it for all, the prompts of 16 138 tokens 577 -> 587).
        if (last - piece < 8) {
#pragma unroll 4
            for (uint32_t k = piece; k <= last; ++k) {
                const float m = ms[slot(k)], f = m == -INFINITY ? 0.0f : exp2_approx(m - M);
                const float4 v = *reinterpret_cast<const float4 *>(os + slot(k));
                L = fmaf(ls[slot(k)], f, L);
                acc.x = fmaf(v.x, f, acc.x);
                acc.y = fmaf(v.y, f, acc.y);
                acc.z = fmaf(v.z, f, acc.z);
                acc.w = fmaf(v.w, f, acc.w);
            }
        } else {
            for (uint32_t k0 = piece; k0 <= last; k0 += 32) {
                const uint32_t k = min(k0 + lane, last), many = min(32u, last - k0 + 1);
                const float m = ms[slot(k)], mine = m == -INFINITY ? 0.0f : exp2_approx(m - M);  // (a part to a lane)
                if (lane < many) L = fmaf(ls[slot(k)], mine, L);
#pragma unroll 8
                for (uint32_t e = 0; e < many; ++e) {
                    const float4 v = *reinterpret_cast<const float4 *>(os + slot(k0 + e));
                    const float f = __shfl_sync(0xffffffffu, mine, e);
                    acc.x = fmaf(v.x, f, acc.x);
                    acc.y = fmaf(v.y, f, acc.y);
                    acc.z = fmaf(v.z, f, acc.z);
                    acc.w = fmaf(v.w, f, acc.w);
                }
            }
            for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const uint32_t token = row_token(l, r);
        const size_t to = ((size_t)(n.t0 + token) * hq + n.kh * l.group + r - token * l.group) * D + 4 * lane;
        if (HALF) *reinterpret_cast<uint2 *>(static_cast<__half *>(o) + to) = make_uint2(pack_h2(acc.x * inv, acc.y * inv), pack_h2(acc.z * inv, acc.w * inv));
        else *reinterpret_cast<float4 *>(static_cast<float *>(o) + to) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}

// What both operators ask of a run beside its pool; the run's view for the kernels.
int32_t packed_view(brasa_ctx *ctx, const char *who, const brasa_paged_kv &pg, const brasa_packed_run &run, uint32_t hq, uint32_t hkv, PackedView *out) {
    BRASA_REQUIRE(ctx, (uint64_t)pg.max_pages * PAGE < 1ull << 31, "%s: max_pages for 2^31 positions or more", who);
    BRASA_TRY(brasa_check_paged(ctx, pg, hq, hkv));
    BRASA_REQUIRE(ctx, hq > 0, "%s: no heads", who);
    BRASA_REQUIRE(ctx, run.tokens >= 1 && run.longest >= 1, "%s: empty run", who);
    BRASA_REQUIRE(ctx, run.starts.offset % 4 == 0 && arg_fits(run.starts, ((uint64_t)pg.seqs + 1) * 4), "%s: starts too small or misaligned", who);
    *out = PackedView{(const int32_t *)arg_ptr(pg.table), (const uint32_t *)arg_ptr(pg.lens), (const uint32_t *)arg_ptr(run.starts), pg.seqs, pg.max_pages,
                      pg.num_pages, run.tokens, run.longest, hkv};
    return BRASA_OK;
}

}  // namespace

extern "C" {

int32_t brasa_k_qk_norm_rope_store_packed(brasa_cmd *cmd, brasa_arg q, brasa_arg k, brasa_arg v, brasa_arg q_norm, brasa_arg k_norm, brasa_arg rope_cos,
                                          brasa_arg rope_sin, float eps, brasa_paged_kv pg, brasa_packed_run run, brasa_arg q_out, uint32_t hq, uint32_t hkv) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    PackedView p;
    BRASA_TRY(packed_view(ctx, "qk_norm_rope_store_packed", pg, run, hq, hkv, &p));
    const uint64_t nq = (uint64_t)run.tokens * hq * 512, nkv = (uint64_t)run.tokens * hkv * 512;
    BRASA_REQUIRE(ctx, arg_fits(q, nq) && arg_fits(q_out, nq) && arg_fits(k, nkv) && arg_fits(v, nkv), "qk_norm_rope_store_packed: q, k, v or q_out too small");
    BRASA_REQUIRE(ctx, arg_fits(q_norm, 512) && arg_fits(k_norm, 512), "qk_norm_rope_store_packed: norm weights too small");
    const uint64_t table_bytes = (uint64_t)pg.max_pages * PAGE * 64 * 4;
    BRASA_REQUIRE(ctx, arg_fits(rope_cos, table_bytes) && arg_fits(rope_sin, table_bytes), "qk_norm_rope_store_packed: RoPE tables shorter than max_pages pages");
    for (const brasa_arg *a : {&q, &k, &v, &q_norm, &k_norm, &rope_cos, &rope_sin, &q_out})
        BRASA_REQUIRE(ctx, a->offset % 16 == 0, "qk_norm_rope_store_packed: misaligned buffer");
    // (in place every warp writes the rows that it has read)
    const uint64_t pool = brasa_kv_bytes(pg.kv, (uint64_t)pg.num_pages * PAGE * hkv * 128), table = (uint64_t)pg.seqs * pg.max_pages * 4, seqs = (uint64_t)pg.seqs * 4;
    const bool in_place = q.buf == q_out.buf && q.offset == q_out.offset;
    const bool over = any_overlap({{q_out, nq}, {pg.kpool, pool}, {pg.vpool, pool}}, {{k, nkv}, {v, nkv}, {q_norm, 512}, {k_norm, 512}, {rope_cos, table_bytes},
                                                                                     {rope_sin, table_bytes}, {run.starts, seqs + 4}, {pg.table, table}, {pg.lens, seqs}}) ||
                      any_overlap({{q, nq}, {q_out, nq}}, {{pg.kpool, pool}, {pg.vpool, pool}}) || arg_overlap(pg.kpool, pool, pg.vpool, pool) ||
                      (!in_place && arg_overlap(q, nq, q_out, nq));
    BRASA_REQUIRE(ctx, !over, "qk_norm_rope_store_packed: q_out (unless it is q) and the pools must overlap neither one another nor what is read");
    const uint32_t per_tok = (hq + 2 * hkv + STORE_ROWS - 1) / STORE_ROWS;
    const uint64_t warps = (uint64_t)run.tokens * per_tok;
    BRASA_REQUIRE(ctx, warps <= 1ull << 33, "qk_norm_rope_store_packed: more than 2^35 rows");
    const dim3 grid((uint32_t)((warps + 7) / 8));
#define STORE_PACKED(KVT)                                                                                                                                       \
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, qk_norm_rope_store_packed_kernel<KVT>, grid, dim3(256), 0, (const float *)arg_ptr(q), (const float *)arg_ptr(k), \
                                           (const float *)arg_ptr(v), (const float *)arg_ptr(q_norm), (const float *)arg_ptr(k_norm),                           \
                                           (const float *)arg_ptr(rope_cos), (const float *)arg_ptr(rope_sin), arg_ptr(pg.kpool), arg_ptr(pg.vpool), p,          \
                                           (float *)arg_ptr(q_out), hq, eps, per_tok, warps))
    if (pg.kv == BRASA_KV_F32) STORE_PACKED(BRASA_KV_F32);
    else if (pg.kv == BRASA_KV_F16) STORE_PACKED(BRASA_KV_F16);
    else STORE_PACKED(BRASA_KV_Q8_0);
#undef STORE_PACKED
    return brasa_post_launch(cmd, "qk_norm_rope_store_packed");
}

int32_t brasa_k_attention_packed(brasa_cmd *cmd, brasa_arg q, brasa_paged_kv pg, brasa_packed_run run, brasa_arg o, uint32_t hq, uint32_t hkv, int32_t precision) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    PackedView p;
    BRASA_TRY(packed_view(ctx, "attention_packed", pg, run, hq, hkv, &p));
    BRASA_REQUIRE(ctx, precision == BRASA_PREFILL_F16 || precision == BRASA_PREFILL_F32, "attention_packed: unknown precision %d", precision);
    const bool half = precision == BRASA_PREFILL_F16;
    const uint64_t n = (uint64_t)run.tokens * hq * D;
    BRASA_REQUIRE(ctx, arg_fits(q, n * 4) && arg_fits(o, n * (half ? 2 : 4)), "attention_packed: q or o too small");
    BRASA_REQUIRE(ctx, q.offset % 16 == 0 && o.offset % 16 == 0, "attention_packed: misaligned buffer");
    const uint64_t pool = brasa_kv_bytes(pg.kv, (uint64_t)pg.num_pages * PAGE * hkv * 128), seqs = (uint64_t)pg.seqs * 4;
    const bool over = any_overlap({{o, n * (half ? 2 : 4)}}, {{q, n * 4}, {pg.kpool, pool}, {pg.vpool, pool}, {pg.table, seqs * pg.max_pages}, {pg.lens, seqs}, {run.starts, seqs + 4}});
    BRASA_REQUIRE(ctx, !over, "attention_packed: o must not overlap what is read");
    BRASA_REQUIRE(ctx, (uint64_t)run.tokens * (hq / hkv) < 1ull << 31, "attention_packed: more than 2^31 rows of a key head's group");
    const float scale = 1.0f / sqrtf((float)D);
    // Sequences of many rows go to the tensor-core kernel where there is one (16-bit products) and the call can have any. What is neither an f16 cache nor 16-bit
    // products of an 8-bit one is computed in 32 bits.
    const uint32_t G = hq / hkv, sms = ctx->sm_count;
    const bool f32 = pg.kv == BRASA_KV_F32 || (pg.kv == BRASA_KV_Q8_0 && !half);
    const bool tc = half && !f32 && (uint64_t)run.longest * G >= PACKED_TC_MIN_ROWS && (uint64_t)pg.num_pages * PAGE < 1ull << 31;
    const uint32_t blocks = sms * (f32 ? 1 : FEW_BLOCKS);
    // the workspace: parts of either kernel's items, then what they belong to
    const size_t few_floats = 2 * (size_t)(FEW_BLOCKS * sms) * packed_part_floats(FEW_ROWS), tc_floats = 2 * (size_t)sms * packed_part_floats(PACKED_TC_ROWS);
    BRASA_TRY(brasa_workspace(ctx, (void **)&ctx->packed_work, &ctx->packed_work_bytes, (few_floats + tc_floats) * sizeof(float) + (FEW_BLOCKS + 1) * sms * sizeof(PackedNote)));
    float *few_part = (float *)ctx->packed_work, *tc_part = few_part + few_floats;
    PackedNote *few_notes = (PackedNote *)(tc_part + tc_floats), *tc_notes = few_notes + FEW_BLOCKS * sms;
    if (tc) BRASA_TRY(brasa_packed_tc_launch(cmd, p, pg.kv, (const float *)arg_ptr(q), arg_ptr(pg.kpool), arg_ptr(pg.vpool), arg_ptr(o), tc_part, tc_notes, hq, scale));
    const FewParams f{packed_line(p, G, FEW_ROWS, 6, 1, 1, 3, 1, tc ? PACKED_TC_MIN_ROWS - 1 : UINT32_MAX), (const float *)arg_ptr(q), arg_ptr(pg.kpool), arg_ptr(pg.vpool), arg_ptr(o), few_part,
                      few_notes, hq, scale, tc ? 1u : 0u};
    void (*kernel)(FewParams);
    size_t smem = F32_SMEM;
    if (f32) {
        kernel = pg.kv == BRASA_KV_Q8_0 ? attn_packed_f32_kernel<BRASA_KV_Q8_0, false> : half ? attn_packed_f32_kernel<BRASA_KV_F32, true> : attn_packed_f32_kernel<BRASA_KV_F32, false>;
    } else if (pg.kv == BRASA_KV_Q8_0) {
        kernel = attn_packed_few_kernel<BRASA_KV_Q8_0, true>;
        smem = FewStage<BRASA_KV_Q8_0>::STAGES * few_stage_bytes<BRASA_KV_Q8_0>();
    } else {
        kernel = half ? attn_packed_few_kernel<BRASA_KV_F16, true> : attn_packed_few_kernel<BRASA_KV_F16, false>;
        smem = FewStage<BRASA_KV_F16>::STAGES * few_stage_bytes<BRASA_KV_F16>();
    }
    BRASA_TRY(brasa_smem_optin(ctx, (const void *)kernel, smem));
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, kernel, dim3(blocks), dim3(f32 ? F32_THREADS : 128), smem, f));
    BRASA_TRY(brasa_post_launch(cmd, f32 ? "attn_packed_f32" : "attn_packed_few"));
    const PackedParts tc_parts{tc_part, tc_notes, tc ? sms : 0u, PACKED_TC_ROWS, 4}, few_parts{few_part, few_notes, blocks, FEW_ROWS, 1};
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, half ? attn_packed_merge_kernel<true> : attn_packed_merge_kernel<false>, dim3((tc ? 4 * sms : 0) + blocks), dim3(256), 0, tc_parts,
                                           few_parts, (void *)arg_ptr(o), hq, packed_line(p, G, FEW_ROWS, 0, 0, 0, 0, 0, 0)));
    return brasa_post_launch(cmd, "attn_packed_merge");
}

}  // extern "C"
