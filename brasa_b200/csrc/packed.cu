// Norm, RoPE and store, and attention, of a packed run: any number of new tokens per sequence over the paged pool.
#include <math.h>

#include "packed_tc.h"

using namespace brasa_dev;

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE;
constexpr int D = 128, TS = D + 4;

// y = x / sqrt(mean x^2 + eps) * w of rows of q and k, rotated by the token's own position (pairs i, i + 64), and the store of k and v. Bound by memory: q read
// and written, k and v read, the cache's rows written. A warp takes four rows of a token (a lane four dims of each, so that a row is one
// request and a pair's other half lies sixteen lanes on), asks for all of them first and finds the token's sequence, position and page meanwhile.
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

// One block per token and key head: the group's rows against 64 keys at a time, K and V as f32 in shared memory, a running maximum, sum
// and output per row.
template <int KV, bool HALF_OUT>
__global__ void __launch_bounds__(128) attn_packed_rows_kernel(const float *q, const uint8_t *kpool, const uint8_t *vpool, PackedView p, void *o, uint32_t hq,
                                                               float scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr uint32_t KEYS = 64;
    __shared__ __align__(16) float ts[KEYS * TS], qs[8 * D], ps[8 * KEYS];
    __shared__ float ms[8], ls[8], alpha[8];
    const uint32_t t = blockIdx.x, kh = blockIdx.y, hkv = p.hkv, G = hq / hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t seq, pos;
    if (!packed_row(p, t, lane, seq, pos) || pos / PAGE >= p.max_pages) return;
    const uint32_t nkeys = pos + 1;
    for (uint32_t i = tid; i < G * D; i += 128) qs[i] = q[((size_t)t * hq + kh * G) * D + i];
    if (tid < 8) {
        ms[tid] = -INFINITY;
        ls[tid] = 0.0f;
    }
    float acc[8];
    for (int g = 0; g < 8; ++g) acc[g] = 0.0f;
    auto load = [&](const uint8_t *pool, uint32_t key0) {
        for (uint32_t i = tid; i < KEYS * (D / 8); i += 128) {
            const uint32_t key = key0 + i / (D / 8), v8 = i % (D / 8);
            const int32_t page = key < nkeys ? packed_page(p, seq, key) : -1;
            float v[8] = {};
            if (page >= 0) tile_load8<KV>(pool + (((size_t)page * PAGE + key % PAGE) * hkv + kh) * KvRow<KV>::BYTES, (int)(v8 * 8), v);
            for (int j = 0; j < 8; ++j) ts[(i / (D / 8)) * TS + v8 * 8 + j] = v[j];
        }
    };
    for (uint32_t key0 = 0; key0 < nkeys; key0 += KEYS) {
        load(kpool, key0);
        __syncthreads();
        const uint32_t key = key0 + (tid & 63);
        const bool there = key < nkeys && packed_page(p, seq, key) >= 0;
        for (uint32_t g = tid >> 6; g < G; g += 2) {
            float a = 0.0f;
            for (int d = 0; d < D; ++d) a = fmaf(qs[g * D + d], ts[(tid & 63) * TS + d], a);
            ps[g * KEYS + (tid & 63)] = there ? a * scale : -INFINITY;
        }
        __syncthreads();
        load(vpool, key0);
        for (uint32_t g = warp; g < G; g += 4) {
            const float s0 = ps[g * KEYS + lane], s1 = ps[g * KEYS + 32 + lane];
            float m = fmaxf(s0, s1);
            for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float before = ms[g], now = fmaxf(before, m);
            const float p0 = s0 == -INFINITY ? 0.0f : expf(s0 - now), p1 = s1 == -INFINITY ? 0.0f : expf(s1 - now);
            float l = p0 + p1;
            for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            ps[g * KEYS + lane] = p0;
            ps[g * KEYS + 32 + lane] = p1;
            __syncwarp();
            if (lane == 0) {
                const float a = before == -INFINITY ? 0.0f : expf(before - now);
                alpha[g] = a;
                ls[g] = ls[g] * a + l;
                ms[g] = now;
            }
        }
        __syncthreads();
        for (uint32_t g = 0; g < G; ++g) {
            float a = acc[g] * alpha[g];
            for (uint32_t j = 0; j < KEYS; ++j) a = fmaf(ps[g * KEYS + j], ts[j * TS + tid], a);
            acc[g] = a;
        }
        __syncthreads();
    }
    for (uint32_t g = 0; g < G; ++g) {
        const float r = ls[g] == 0.0f ? 0.0f : acc[g] / ls[g];
        const size_t at = ((size_t)t * hq + kh * G + g) * D + tid;
        if (HALF_OUT) static_cast<__half *>(o)[at] = __float2half_rn(r);
        else static_cast<float *>(o)[at] = r;
    }
}

// ---- few rows against many keys: the cache's bytes are the work ------------------------------------------------------------------
// Four warps, 64 keys at a time through a ring of cp.async stages. An item's up to 64 rows are one to four tiles of 16 for mma.sync m16n8k16;
// with one tile the warps share the keys (a page each), with two they go in pairs, with more every warp has a tile of its own. Each warp keeps a
// running maximum, sum and output (the maximum moves only when a score passes it by 2^8), the warps meet at the item's end. The 16 keys of a
// warp's step are one page: a page that is none is skipped, and rows of the cache that the sequence has not reached are never loaded.
// HALF: one f16 term of q * scale and of P, 8-bit rows as f16(d * code): what the F16 precision says. Otherwise q and P enter as two terms, hi + lo
// (2^-22 of the value), and an f16 cache's rows as they are.
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
constexpr uint32_t FEW_ROWS = 64, FEW_KEYS = 64;
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
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
__global__ void __launch_bounds__(128) attn_packed_few_kernel(const __grid_constant__ FewParams p) {
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
        // ---- copies of 64 keys: pages one chunk ahead, what the item's last row does not see as zeros ----
        const int32_t *table = p.l.v.table + (size_t)it.seq * p.l.v.max_pages;
        const size_t page_bytes = (size_t)PAGE * hkv * ROW;
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
                if (!Q8) {
                    const uint32_t r = tid >> 4, c = tid & 15;
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t row = 8 * k + r;
                        const bool ok = pg[k >> 1] >= 0 && 64 * j + row < nkeys;
                        const size_t at = (ok ? (size_t)pg[k >> 1] : 0) * page_bytes + ((row & 15) * hkv + it.kh) * ROW + 16 * c;
                        const uint32_t to = stage + row * 256 + ((c ^ (row & 7)) << 4);
                        cp_zfill16(to, p.kpool + at, ok);
                        cp_zfill16(to + V_AT, p.vpool + at, ok);
                    }
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 9; ++k) {
                        const uint32_t i = tid + 128 * k, row = i / 17, c = i % 17;
                        if (i >= FEW_KEYS * 17) break;
                        const int32_t page = row < 32 ? (row < 16 ? pg[0] : pg[1]) : (row < 48 ? pg[2] : pg[3]);
                        const bool ok = page >= 0 && 64 * j + row < nkeys;
                        const size_t at = (ok ? (size_t)page : 0) * page_bytes + ((row & 15) * hkv + it.kh) * ROW + 8 * c;
                        cp_zfill8(stage + row * S::K_PITCH + 8 * c, p.kpool + at, ok);
                        cp_zfill8(stage + V_AT + row * S::V_PITCH + 8 * c, p.vpool + at, ok);
                    }
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
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t r = rt * 16 + g + 8 * h;
            const bool live = active && r < rows;
            const uint32_t token = live ? row_token(p.l, r) : 0, head = live ? r - token * G : 0;
            seen[h] = live ? it.past + token0 + token + 1 : 0;
            const float *src = p.q + ((size_t)(t0 + token) * p.hq + it.kh * G + head) * D;
#pragma unroll
            for (uint32_t ks = 0; ks < 8; ++ks) {
                float2 a = make_float2(0.0f, 0.0f), b = a;
                const uint32_t d0 = Q8 ? 32 * (ks >> 1) + 8 * tq + 4 * (ks & 1) : 16 * ks + 2 * tq, d1 = Q8 ? d0 + 2 : d0 + 8;
                if (live) {
                    a = *reinterpret_cast<const float2 *>(src + d0);
                    b = *reinterpret_cast<const float2 *>(src + d1);
                }
                const float f = HALF ? p.scale : 1.0f;
                terms_h2<HALF>(a.x * f, a.y * f, qh[ks][h], ql[ks][h]);
                terms_h2<HALF>(b.x * f, b.y * f, qh[ks][h + 2], ql[ks][h + 2]);
            }
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(seen[0], seen[1]));  // keys that any row of the tile sees
        const float c = HALF ? LOG2E : p.scale * LOG2E;
        float m[2] = {-INFINITY, -INFINITY}, l[4] = {0.0f, 0.0f, 0.0f, 0.0f}, o[16][4];  // (l: a column of ones beside V, so that it sums the very P)
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
#pragma unroll
                        for (uint32_t ks = 0; ks < 8; ks += 2) {
                            uint32_t b[4];
                            ldsm_x4(b, kt + row * 256 + (((2 * ks + (lane >> 3)) ^ (row & 7)) << 4));
                            mma_f16(s[t], qh[ks], b[0], b[1]);
                            if (!HALF) mma_f16(s[t], ql[ks], b[0], b[1]);
                            mma_f16(s[t], qh[ks + 1], b[2], b[3]);
                            if (!HALF) mma_f16(s[t], ql[ks + 1], b[2], b[3]);
                        }
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
                // ---- P = 2^(s - m) ----
                uint32_t ph[4], pl[4];
                bool moved = false;
                float back[2] = {1.0f, 1.0f};
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    float x[4], top = -INFINITY;
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t key = key0 + 8 * (e >> 1) + 2 * tq + (e & 1);
                        x[e] = key < seen[h] ? s[e >> 1][2 * h + (e & 1)] * c : -INFINITY;
                        top = fmaxf(top, x[e]);
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (top > m[h] + SLACK || (m[h] == -INFINITY && top > -INFINITY)) {
                        moved = true;
                        back[h] = m[h] == -INFINITY ? 0.0f : exp2_approx(m[h] - top);
                        m[h] = top;
                    }
                    const float ref = m[h] == -INFINITY ? 0.0f : m[h];
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
                mma_f16(l, ph, ones, ones);
                if (!HALF) mma_f16(l, pl, ones, ones);
                if (!Q8) {
#pragma unroll
                    for (uint32_t n = 0; n < 16; n += 2) {
                        uint32_t b[4];
                        ldsm_x4_t(b, vt + vrow * 256 + (((n + (lane >> 4)) ^ (vrow & 7)) << 4));
                        mma_f16(o[n], ph, b[0], b[1]);
                        if (!HALF) mma_f16(o[n], pl, b[0], b[1]);
                        mma_f16(o[n + 1], ph, b[2], b[3]);
                        if (!HALF) mma_f16(o[n + 1], pl, b[2], b[3]);
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
                sums[warp][0][g + 8 * h] = m[h];
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
        __syncthreads();
        const bool whole = j0 == 0 && j1 == it.tiles;
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
        if (j1 < it.tiles || !line_next(p.l, it)) break;
    }
    if (tid == 0) p.notes[blockIdx.x] = note;
    if (p.late_wait) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// What either kernel left of the items that several blocks worked on.
struct PackedParts {
    const float *part;
    const PackedNote *notes;
    uint32_t pieces, rows_item, spread;  // blocks, rows of an item, merging blocks to a piece
};
// Such an item is the work of the piece that began and left it open, each of that piece's `spread` blocks with every spread * 8-th row: the sum of 2^(m - M) O over
// that of 2^(m - M) l, in the order of the keys.
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
    uint32_t last = piece + 1;  // the piece that ends the item
    while (last + 1 < p.pieces && !notes[last].closes) ++last;
    for (uint32_t r = share * 8 + warp; r < n.rows; r += p.spread * 8) {
        const float *ms = part + rows_item * D + r, *ls = ms + rows_item, *os = part + (size_t)r * D + 4 * lane;
        // (slot 2 b + 1 is what piece b left open, slot 2 k piece k's share of an item that began before it)
        auto slot = [&](uint32_t k) { return (k == piece ? 2 * (size_t)k + 1 : 2 * (size_t)k) * step; };
        float M = -INFINITY;
        for (uint32_t k = piece + lane; k <= last; k += 32) M = fmaxf(M, ms[slot(k)]);
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        float L = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const uint32_t token = row_token(l, r);
        const size_t to = ((size_t)(n.t0 + token) * hq + n.kh * l.group + r - token * l.group) * D + 4 * lane;
        if (HALF) *reinterpret_cast<uint2 *>(static_cast<__half *>(o) + to) = make_uint2(pack_h2(acc.x * inv, acc.y * inv), pack_h2(acc.z * inv, acc.w * inv));
        else *reinterpret_cast<float4 *>(static_cast<float *>(o) + to) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}

// What both operators ask of a run beside its pool; the run's view for the kernels.
int32_t packed_view(brasa_ctx *ctx, const char *who, const brasa_paged_kv &pg, const brasa_packed_run &run, uint32_t hq, uint32_t hkv, PackedView *out) {
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
    BRASA_REQUIRE(ctx, run.tokens < 1u << 31 && hkv <= 65535, "attention_packed: more than 2^31 tokens or 65 535 key heads");
    BRASA_REQUIRE(ctx, (uint64_t)run.tokens * (hq / hkv) < 1ull << 31, "attention_packed: more than 2^31 rows of a key head's group");
    const float scale = 1.0f / sqrtf((float)D);
    if (pg.kv == BRASA_KV_F16 || (pg.kv == BRASA_KV_Q8_0 && half)) {
        // Sequences of many rows go to the tensor-core kernel where there is one (16-bit products) and the call can have any.
        const uint32_t G = hq / hkv, sms = ctx->sm_count, blocks = sms * 2;
        const bool tc = half && (uint64_t)run.longest * G >= PACKED_TC_MIN_ROWS && (uint64_t)pg.num_pages * PAGE < 1ull << 31;
        // the workspace: parts of either kernel's items, then what they belong to
        const size_t few_floats = 2 * (size_t)blocks * packed_part_floats(FEW_ROWS), tc_floats = 2 * (size_t)sms * packed_part_floats(PACKED_TC_ROWS);
        BRASA_TRY(brasa_workspace(ctx, (void **)&ctx->packed_work, &ctx->packed_work_bytes, (few_floats + tc_floats) * sizeof(float) + (blocks + sms) * sizeof(PackedNote)));
        float *few_part = (float *)ctx->packed_work, *tc_part = few_part + few_floats;
        PackedNote *few_notes = (PackedNote *)(tc_part + tc_floats), *tc_notes = few_notes + blocks;
        if (tc) BRASA_TRY(brasa_packed_tc_launch(cmd, p, pg.kv, (const float *)arg_ptr(q), arg_ptr(pg.kpool), arg_ptr(pg.vpool), arg_ptr(o), tc_part, tc_notes, hq, scale));
        FewParams f{packed_line(p, G, FEW_ROWS, 6, 1, 1, 3, 1, tc ? PACKED_TC_MIN_ROWS - 1 : UINT32_MAX), (const float *)arg_ptr(q), arg_ptr(pg.kpool), arg_ptr(pg.vpool), arg_ptr(o), few_part,
                    few_notes, hq, scale, tc ? 1u : 0u};
        void (*const kernel)(FewParams) = pg.kv == BRASA_KV_Q8_0 ? attn_packed_few_kernel<BRASA_KV_Q8_0, true>
                                          : half ? attn_packed_few_kernel<BRASA_KV_F16, true> : attn_packed_few_kernel<BRASA_KV_F16, false>;
        const size_t smem = pg.kv == BRASA_KV_Q8_0 ? FewStage<BRASA_KV_Q8_0>::STAGES * few_stage_bytes<BRASA_KV_Q8_0>() : FewStage<BRASA_KV_F16>::STAGES * few_stage_bytes<BRASA_KV_F16>();
        BRASA_TRY(brasa_smem_optin(ctx, (const void *)kernel, smem));
        BRASA_CUDA(ctx, brasa_launch_dependent(ctx, kernel, dim3(blocks), dim3(128), smem, f));
        BRASA_TRY(brasa_post_launch(cmd, "attn_packed_few"));
        const PackedParts tc_parts{tc_part, tc_notes, tc ? sms : 0u, PACKED_TC_ROWS, 4}, few_parts{few_part, few_notes, blocks, FEW_ROWS, 1};
        BRASA_CUDA(ctx, brasa_launch_dependent(ctx, half ? attn_packed_merge_kernel<true> : attn_packed_merge_kernel<false>, dim3((tc ? 4 * sms : 0) + blocks), dim3(256), 0, tc_parts,
                                               few_parts, (void *)arg_ptr(o), hq, packed_line(p, G, FEW_ROWS, 0, 0, 0, 0, 0, 0)));
        return brasa_post_launch(cmd, "attn_packed_merge");
    }
#define ATTN_PACKED(KVT)                                                                                                                                  \
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, half ? attn_packed_rows_kernel<KVT, true> : attn_packed_rows_kernel<KVT, false>, dim3(run.tokens, hkv), dim3(128), 0, \
                                           (const float *)arg_ptr(q), (const uint8_t *)arg_ptr(pg.kpool), (const uint8_t *)arg_ptr(pg.vpool), p, (void *)arg_ptr(o), hq, scale))
    if (pg.kv == BRASA_KV_F32) ATTN_PACKED(BRASA_KV_F32);
    else if (pg.kv == BRASA_KV_F16) ATTN_PACKED(BRASA_KV_F16);
    else ATTN_PACKED(BRASA_KV_Q8_0);
#undef ATTN_PACKED
    return brasa_post_launch(cmd, "attn_packed_rows");
}

}  // extern "C"
