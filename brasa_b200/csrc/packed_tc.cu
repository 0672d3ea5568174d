// Attention of a packed run's sequences of many rows on the 5th-generation tensor cores (F16 precision, f16 caches), over pages.
//
// An item is 256 rows of one sequence against one key head, in two tiles of 128; a row is a token and a head of the group, so that short
// prompts of grouped heads fill their tiles and all heads of a group share K and V. Per tile of 128 keys and row tile there are two products of
// 128^3: S = Q K^T into tensor memory, O += P V with P read out of tensor memory, over the columns that S had. Two threads hold a row, 64 scores
// each: warps 0-7 tile A, 8-15 tile B; warp 16 issues the products, warp 17 the copies. The order on the tensor core is P V of A, S of
// A's next keys, P V of B, S of B's next, so that one tile's products run while the other's probabilities are formed.
// K and V tiles are eight pages each, two boxes of 16 positions x 64 dims a page (cp.async.bulk.tensor, 128-byte swizzle), through a ring of four
// 32 KB slots. Rows of the cache behind the item's last position may hold anything: such scores are replaced before they count, and V's rows,
// which enter P V with a weight of zero, are written as zeros by the copying warp instead of copied.
// What bounds it: the tensor core, 2 048 cycles per tile of keys, and as many cycles of exponentials (16 a clock).
#include <math.h>

#include "packed_tc.h"
#include "tc_device.cuh"

using namespace brasa_dev;

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE, D = 128, WAIT_LIMIT = 1u << 20, TILE_BYTES = 128 * 128 * 2, SLOTS = 4, ROWS = PACKED_TC_ROWS;
constexpr uint32_t SOFTMAX_WARPS = 16, MMA_WARP = 16, COPY_WARP = 18, THREADS = 608;  // (one MMA warp for each row tile)

struct PackedMaps {
    CUtensorMap k, v;
};
struct PackedTcParams {
    PackedLine l;
    const float *q;
    const uint8_t *vpool;
    __half *o;
    float *part;
    PackedNote *notes;
    uint32_t hq;
    float scale;
    uint32_t *status;
};

// byte offset of the 16-byte piece of columns [c, c + 8) of row r in a swizzled 128 x 128 tile of 16-bit values
__device__ __forceinline__ uint32_t tile_piece(uint32_t r, uint32_t c) {
    return (c >> 6) * 16384 + (r >> 3) * 1024 + (r & 7) * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t v[32]) {  // (the caller waits for its loads)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t v[8]) {  // (the caller waits for its stores)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t v[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t v[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// adds both halves of a pair to a sum of 32 bits: the sum of the weights that the product reads, rounded as they are
__device__ __forceinline__ void add_halves(uint32_t pair, float &a, float &b) {
    asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tadd.rn.f32.f16 %0, x, %0;\n\tadd.rn.f32.f16 %1, y, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(pair));
}

__global__ void __launch_bounds__(THREADS, 1) attn_packed_tc_kernel(const __grid_constant__ PackedMaps maps, const __grid_constant__ PackedTcParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *ring = smem + 2 * TILE_BYTES;
    __shared__ uint64_t full[SLOTS], freed[SLOTS], q_full[2], s_ready[2], p_ready[2][2], o_done[2], turn[2];
    __shared__ uint32_t tmem_base_s, abort_s, there_s[8];  // (there: of the last key tiles, which of their eight pages are pages)
    __shared__ float pair[2][2][128];                      // [row tile][half of the keys][row]: largest score; at the end the sum of the weights
    __shared__ PackedPieces pieces;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.l.group, hkv = p.l.v.hkv;

    if (tid == 0) {
        for (uint32_t i = 0; i < SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&freed[i], 2);  // by either row tile's products
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 8);  // one arrival per softmax warp of the row tile
            mbar_init(&s_ready[i], 1);
            mbar_init(&p_ready[i][0], 8);
            mbar_init(&p_ready[i][1], 8);
            mbar_init(&turn[i], 8);  // of the other row tile's warps
            mbar_init(&o_done[i], 1);
        }
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {  // tensor memory: S, then P over the first half of either 64 keys, of A in [0, 128), of B in [128, 256); O of A in [256, 384), of B in [384, 512)
        const uint32_t ncols = 512;
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(ncols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // launched as a programmatic dependent: what the kernels before this one wrote (q, the cache, its tables) is touched after the wait
    pdl_wait();
    pdl_launch();
    const uint32_t tmem = tmem_base_s;
    volatile uint32_t *abort_flag = &abort_s;
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        for (uint32_t it = 0; it < WAIT_LIMIT; ++it) {
            if (tc_mbar_try(bar, parity)) return true;
            if (*abort_flag) return false;
        }
        atomicExch(p.status, 7u);
        *abort_flag = 1;
        return false;
    };
    auto all_wait = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (smem_u32(smem) & 1023) {  // (the swizzle counts from there)
        if (tid == 0) atomicExch(p.status, 8u);
        abort_s = 1;
    }
    const bool work = line_cut<256>(p.l, pieces) && !abort_s;
    // Every role walks through the block's items by itself; they meet at barriers of their own only.
    PackedItem item = pieces.at[0];
    const uint64_t end_first = pieces.at[1].first;
    const uint32_t end_j = pieces.at[1].j;
    if (work && item.j == item.tiles) line_next(p.l, item);
    bool more = work && (item.first < end_first || (item.first == end_first && item.j < end_j));
    auto item_end = [&]() { return item.first == end_first ? end_j : item.tiles; };  // the key tile at which this block's share of the item ends
    auto next_item = [&](PackedItem &it, uint32_t j1) { return j1 == it.tiles && line_next(p.l, it) && (it.first < end_first || (it.first == end_first && end_j > 0)); };
    auto has_b = [&](const PackedItem &it) { return line_tokens(p.l, it) * G > 128; };  // rows in both row tiles
    if (warp == COPY_WARP) {  // ---- K and V, as far ahead of the products as there are slots ----
        bool ok = true;
        uint32_t loads = 0;  // tiles copied so far, K and V apart
#pragma unroll 1
        while (more && ok) {
            const uint32_t j0 = item.j, j1 = item_end(), nkeys = line_keys(p.l, item);
            const int32_t *table = p.l.v.table + (size_t)item.seq * p.l.v.max_pages;
            auto page_at = [&](uint32_t i) { return (uint64_t)16 * i < nkeys ? table[i] : -1; };  // as the table has it, -1 where nothing is seen
            int32_t now = page_at(8 * j0 + lane), ahead = page_at(8 * j0 + 32 + lane);           // the pages of four tiles, and of the next four
            for (uint32_t t = lane; t < line_tokens(p.l, item); t += 32)  // the item's queries on their way into L2
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.q + ((size_t)(item.t0 + item.part * p.l.item_tokens + t) * p.hq + item.kh * G) * D), "r"(G * D * 4) : "memory");
            for (uint32_t j = j0; j < j1 && ok; ++j) {
                const uint32_t k = (j - j0) & 3, half = lane & 1, i = (lane >> 1) & 7;  // lanes 2 i and 2 i + 1 take the halves of page i
                if (j > j0 && k == 0) {
                    now = ahead;
                    ahead = page_at(8 * j + 32 + lane);
                }
                int32_t page = __shfl_sync(0xffffffffu, now, 8 * k + i);
                if ((uint32_t)page >= p.l.v.num_pages) page = -1;
                const uint32_t there = __ballot_sync(0xffffffffu, (uint32_t)now < p.l.v.num_pages) >> (8 * k) & 255;
                const uint32_t left = nkeys - min(nkeys, 128 * j + 16 * i);  // of the page's positions, those that are seen
                for (uint32_t is_v = 0; is_v < 2; ++is_v, ++loads) {
                    const uint32_t s = loads % SLOTS;
                    if (loads >= SLOTS && !all_wait(&freed[s], ((loads / SLOTS) - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    uint8_t *slot = ring + (size_t)s * TILE_BYTES;
                    const bool whole = page >= 0 && (!is_v || left >= 16);
                    const uint32_t odd = is_v ? __ballot_sync(0xffffffffu, !whole) & 0x5555u : 0u;  // bit 2 i: page i is not copied whole
                    for (uint32_t b = odd; b; b &= b - 1) {  // what is seen of it, and zeros
                        const uint32_t e = (__ffs(b) - 1) >> 1, seen = __shfl_sync(0xffffffffu, page >= 0 ? left : 0u, 2 * e);
                        const int32_t from = __shfl_sync(0xffffffffu, page, 2 * e);
                        uint4 v[8];
#pragma unroll
                        for (uint32_t u = 0; u < 8; ++u) {
                            const uint32_t r = 2 * u + (lane >> 4);
                            v[u] = make_uint4(0, 0, 0, 0);
                            if (r < seen) v[u] = reinterpret_cast<const uint4 *>(p.vpool + (((size_t)from * PAGE + r) * hkv + item.kh) * 256)[lane & 15];
                        }
#pragma unroll
                        for (uint32_t u = 0; u < 8; ++u) *reinterpret_cast<uint4 *>(slot + tile_piece(16 * e + 2 * u + (lane >> 4), 8 * (lane & 15))) = v[u];
                    }
                    if (odd) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    const uint32_t copies = __popc(__ballot_sync(0xffffffffu, whole) & 0xffffu);
                    if (lane == 0) {
                        if (!is_v) there_s[(loads >> 1) & 7] = there;  // (read by whoever sees this tile's scores; the ring is at most four loads ahead)
                        mbar_expect_tx(&full[s], copies * 2048);
                    }
                    __syncwarp();
                    if (whole && lane < 16) tma_load_3d(slot + half * 16384 + i * 2048, is_v ? &maps.v : &maps.k, (int)(half * 64), (int)item.kh, page * (int)PAGE, &full[s]);
                }
            }
            more = next_item(item, j1);
        }
        if (*abort_flag && lane == 0) {  // leaving early: let the copies in flight land before the block's shared memory is handed on
            for (uint32_t k = loads > SLOTS ? loads - SLOTS : 0; k < loads; ++k)
                for (uint32_t it = 0; it < WAIT_LIMIT && !tc_mbar_try(&full[k % SLOTS], (k / SLOTS) & 1); ++it) {}
        }
    } else if (warp == MMA_WARP || warp == MMA_WARP + 1) {  // ---- products of one row tile: the warp waits, one lane issues ----
        const uint32_t idesc_s = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24), idesc_o = idesc_s | (1u << 16);  // f16 operands; V is MN-major
        const uint32_t x = warp - MMA_WARP, st = tmem + 128 * x, ot = tmem + 256 + 128 * x;
        auto landed = [&](uint32_t m) { return all_wait(&full[m % SLOTS], (m / SLOTS) & 1); };
        auto slot = [&](uint32_t m) { return smem_u32(ring + (size_t)(m % SLOTS) * TILE_BYTES); };
        uint32_t loads = 0, done = 0, segs = 0;  // of the items before: tiles copied, key tiles of this row tile, items with this row tile
        bool ok = true;
#pragma unroll 1
        while (more && ok) {
            const uint32_t j0 = item.j, j1 = item_end(), len = j1 - j0;
            const bool both = has_b(item);
            if (x == 1 && !both) {  // no rows: the slots are given back as they come
                for (uint32_t m = loads; ok && m < loads + 2 * len; ++m) {
                    ok = landed(m);
                    if (ok && lane == 0) tc_mbar_arrive(&freed[m % SLOTS]);
                }
            } else {
                const uint32_t q = smem_u32(smem + x * TILE_BYTES);
                ok = all_wait(&q_full[x], segs & 1);
                for (uint32_t j = 0; j <= len && ok; ++j) {
                    const uint32_t mv = loads + 2 * j - 1, mk = loads + 2 * j;
                    ok = (j == 0 || landed(mv)) && (j == len || landed(mk));
                    if (!ok) break;
                    if (j > 0) {  // O += P V of the tile before, in two halves as they come
                        const uint32_t v = slot(mv);
#pragma unroll
                        for (uint32_t e = 0; e < 2 && ok; ++e) {
                            ok = all_wait(&p_ready[x][e], (done + j - 1) & 1);
                            if (!ok) break;
                            if (tc_elect_one()) {
                                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                                for (uint32_t k = 0; k < 4; ++k) {  // 16 keys: 8 columns of P; 32 keys of either half of the tile
                                    const uint32_t ks = 4 * (k >> 1) + 2 * e + (k & 1);
                                    tc_mma_ta(ot, st + 64 * (ks >> 2) + 8 * (ks & 3), tc_desc_mnmajor(v + ks * 2048), idesc_o, (j > 1 || e > 0 || k > 0) ? 1u : 0u);
                                }
                                if (e == 1) tc_commit(&freed[mv % SLOTS]);
                                if (e == 1 && j == len) tc_commit(&o_done[x]);
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                    }
                    if (j < len) {  // S = Q K^T of this tile, over the columns of the P just read
                        if (tc_elect_one()) {
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint32_t k = slot(mk);
#pragma unroll
                            for (uint32_t ks = 0; ks < 8; ++ks) {
                                const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
                                tc_mma(st, tc_desc_kmajor(q + off), tc_desc_kmajor(k + off), idesc_s, ks > 0 ? 1u : 0u);
                            }
                            tc_commit(&s_ready[x]);
                            tc_commit(&freed[mk % SLOTS]);
                        }
                        __syncwarp();
                    }
                }
                done += len;
                ++segs;
            }
            loads += 2 * len;
            more = next_item(item, j1);
        }
        if (*abort_flag) {  // leaving early: the products in flight end before the block's memory is handed on (one commit more to the output's barrier)
            if (tc_elect_one()) tc_commit(&o_done[x]);
            __syncwarp();
            for (uint32_t it = 0; it < 4096 && !tc_mbar_try(&o_done[x], segs & 1); ++it) {}
        }
    } else if (warp < SOFTMAX_WARPS) {  // ---- softmax: two threads per row, 64 keys of every tile each ----
        constexpr float LOG2E = 1.4426950408889634f, SLACK = 5.545177444f;  // 8 ln 2
        const uint32_t x = warp >> 3, h = (warp >> 2) & 1, wrow = (warp & 3) * 32, row = wrow + lane;
        const uint32_t ts = tmem + 128 * x + 64 * h + (wrow << 16), to = tmem + 256 + 128 * x + 64 * h + (wrow << 16);
        const uint32_t both = 2 + 4 * x + (warp & 3);       // named barrier of the two warps that hold these rows
        uint32_t done = 0, segs = 0, turns = 0, tiles0 = 0;  // of the items before: key tiles and items of this row tile, tiles with both; all key tiles
        PackedNote note{};
        // The warp's 32 rows and 64 dims of an item's q: fetched, and when `before` has waited for the last scores of the item before, scaled, rounded to f16 and
        // stored swizzled K-major over that item's (rows past the last are zeros).
        auto bring_q = [&](const PackedItem &it, auto before) -> bool {
            const uint32_t rows = line_tokens(p.l, it) * G;
            const float *q0 = p.q + ((size_t)(it.t0 + it.part * p.l.item_tokens) * p.hq + it.kh * G) * D + 64 * h;
            float4 f[16];
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) {
                const uint32_t r = 128 * x + wrow + 2 * e + (lane >> 4), token = row_token(p.l, r);
                f[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (r < rows) f[e] = reinterpret_cast<const float4 *>(q0 + (token * p.hq + r - token * G) * D)[lane & 15];
            }
            const bool fine = before();
            uint8_t *to_q = smem + x * TILE_BYTES;
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) {
                const __half2 a = __floats2half2_rn(f[e].x * p.scale, f[e].y * p.scale), b = __floats2half2_rn(f[e].z * p.scale, f[e].w * p.scale);
                *reinterpret_cast<uint2 *>(to_q + tile_piece(wrow + 2 * e + (lane >> 4), 64 * h + 8 * ((lane & 15) >> 1)) + 8 * (lane & 1)) =
                    make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(&q_full[x]);
            return fine;
        };
        auto nothing = [] { return true; };
        bool ok = true;
        if (more && (x == 0 || has_b(item))) ok = bring_q(item, nothing);
#pragma unroll 1
        while (more && ok) {
            const uint32_t j0 = item.j, j1 = item_end(), len = j1 - j0, tiles = item.tiles, kh = item.kh, past = item.past + item.part * p.l.item_tokens;
            const uint32_t t0 = item.t0 + item.part * p.l.item_tokens, rows = line_tokens(p.l, item) * G, r = 128 * x + row;
            const bool live = r < rows, pairs = rows > 128, used = x == 0 || pairs;
            const uint32_t seen_all = live ? past + row_token(p.l, r) + 1 : 0;
            const uint32_t nfree = (past + row_token(p.l, 128 * x) + 1) / 128;  // tiles [0, nfree) lie wholly at or below every row's own position
            float m = -INFINITY, mneg = 0.0f, l0 = 0.0f, l1 = 0.0f;
            more = next_item(item, j1);  // (from here on `item` is the next one)
            const bool fetch = more && (x == 0 || has_b(item));
            if (!used) {
                if (fetch) ok = bring_q(item, nothing);
            } else {
#pragma unroll 1
                for (uint32_t j = j0; j < j1; ++j) {
                    auto scores = [&] { return all_wait(&s_ready[x], (done + j - j0) & 1); };  // S of this tile, and with it every product issued before: P V of the tile before
                    if (j + 1 == j1 && fetch) ok = bring_q(item, scores);  // (the next item's queries on the way)
                    else ok = scores();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint32_t v[2][32];
                    tmem_ld32(ts, v[0]);
                    tmem_ld32(ts + 32, v[1]);
                    const uint32_t there = there_s[(tiles0 + j - j0) & 7] >> (4 * h) & 15;  // of the four pages of this thread's keys, those that are pages
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (j >= nfree || there != 15) {
                        const int seen = (int)min(64u, seen_all - min(seen_all, j * 128 + 64 * h));  // of this thread's keys, those the row sees
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (i >= seen || !(there >> (i >> 4) & 1)) v[i >> 5][i & 31] = 0xff800000u;  // -inf: exp2 gives 0
                    }
                    float t[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[i] = fmaxf(__uint_as_float(v[0][2 * i]), __uint_as_float(v[0][2 * i + 1]));
#pragma unroll
                    for (int i = 8; i < 64; i += 2) t[(i >> 1) & 3] = max3(t[(i >> 1) & 3], __uint_as_float(v[i >> 5][i & 31]), __uint_as_float(v[i >> 5][(i & 31) + 1]));
                    float tmax = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
                    pair[x][h][row] = tmax;
                    ok = tc_pair_agree(both, ok);  // (after a wait that gave up, what was read of S counts for nothing)
                    if (!ok) break;
                    tmax = fmaxf(tmax, pair[x][h ^ 1][row]);
                    float rescale = 1.0f;
                    bool move = false;
                    if (tmax > m + SLACK || (m == -INFINITY && tmax != -INFINITY)) {
                        move = m != -INFINITY;
                        rescale = move ? ex2((m - tmax) * LOG2E) : 1.0f;
                        l0 *= rescale;
                        l1 *= rescale;
                        m = tmax;
                        mneg = -m * LOG2E;
                    }
                    if (__any_sync(0xffffffffu, move)) {  // what O holds for the row was accumulated against the old reference
#pragma unroll 1
                        for (uint32_t c = 0; c < 64; c += 8) {
                            uint32_t o[8];
                            tmem_ld8(to + c, o);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * rescale);
                            tmem_st8(to + c, o);
                        }
                    }
                    // The row tiles take turns with the exponentials, A first: side by side both would end late, and both would wait for the tensor core at once.
                    if (pairs) {
                        if (x == 1 || turns > 0) {
                            ok = wait(&turn[x], (turns - (x ^ 1)) & 1);
                            ok = __all_sync(0xffffffffu, ok);
                        }
                        ++turns;
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) {  // 16 keys: 8 columns of P (all of this thread's scores are in registers by now)
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const int k = 16 * c + i;
                            const __half2 e = __floats2half2_rn(ex2(fmaf(__uint_as_float(v[k >> 5][k & 31]), LOG2E, mneg)), ex2(fmaf(__uint_as_float(v[k >> 5][(k & 31) + 1]), LOG2E, mneg)));
                            w[i >> 1] = *reinterpret_cast<const uint32_t *>(&e);
                            add_halves(w[i >> 1], l0, l1);
                        }
                        tmem_st8(ts + 8 * c, w);
                        if (c == 3 && pairs && lane == 0) tc_mbar_arrive(&turn[x ^ 1]);
                        if (c & 1) {  // half of P is there for the product
                            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) tc_mbar_arrive(&p_ready[x][c >> 1]);
                        }
                    }
                }
                done += len;
                // ---- output: O / l, rounded to f16; a part of the item's keys: O, m and l as they are ----
                ok = ok && wait(&o_done[x], segs & 1);
                ok = __all_sync(0xffffffffu, ok);
                ++segs;
                if (ok) pair[x][h][row] = l0 + l1;
                ok = tc_pair_agree(both, ok);
                if (!ok) break;
                const float l = l0 + l1 + pair[x][h ^ 1][row];
                tc_pair_agree(both, ok);  // (both have read: the next item's scores come there)
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (len < tiles) {
                    float *dst = p.part + (size_t)(2 * blockIdx.x + (j0 == 0)) * packed_part_floats(ROWS);
                    if (live && h == 0) {
                        dst[ROWS * D + r] = m * LOG2E;
                        dst[ROWS * D + ROWS + r] = l;
                    }
#pragma unroll 1
                    for (uint32_t c = 0; c < 4; ++c) {
                        uint32_t o[16];
                        tmem_ld16(to + 16 * c, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int g = 0; g < 4; ++g)
                            if (live) reinterpret_cast<uint4 *>(dst + (size_t)r * D + 64 * h)[4 * c + g] = make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
                    }
                } else {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    uint8_t *stage = ring + SLOTS * TILE_BYTES + warp * 2048;  // 32 rows of 32 dims; a piece of 16 bytes goes where no two meet in a bank
#pragma unroll 1
                    for (uint32_t c = 0; c < 2; ++c) {
                        uint32_t o[32], packed[16];
                        tmem_ld32(to + 32 * c, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const __half2 hh = __floats2half2_rn(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                            packed[i >> 1] = *reinterpret_cast<const uint32_t *>(&hh);
                        }
#pragma unroll
                        for (uint32_t g = 0; g < 4; ++g)
                            *reinterpret_cast<uint4 *>(stage + 64 * lane + 16 * (g ^ (lane >> 1 & 3))) = make_uint4(packed[4 * g], packed[4 * g + 1], packed[4 * g + 2], packed[4 * g + 3]);
                        __syncwarp();
#pragma unroll
                        for (uint32_t g = 0; g < 4; ++g) {  // eight rows at a time, 64 bytes of each
                            const uint32_t e = 8 * g + (lane >> 2), re = 128 * x + wrow + e, tk = row_token(p.l, re);
                            const uint4 w = *reinterpret_cast<const uint4 *>(stage + 64 * e + 16 * ((lane & 3) ^ (e >> 1 & 3)));
                            if (re < rows) reinterpret_cast<uint4 *>(p.o + ((size_t)(t0 + tk) * p.hq + kh * G + re - tk * G) * D + 64 * h + 32 * c)[lane & 3] = w;
                        }
                        __syncwarp();
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            }
            tiles0 += len;
            if (len < tiles && j0 == 0) note = PackedNote{1, note.closes, t0, rows, kh};
            if (j0 > 0 && j1 == tiles) note.closes = 1;
        }
        if (tid == 0) p.notes[blockIdx.x] = note;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t ncols = 512;
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(ncols) : "memory");
    }
}

}  // namespace

int32_t brasa_packed_tc_launch(brasa_cmd *cmd, const PackedView &v, const float *q, const uint8_t *kpool, const uint8_t *vpool, void *o, float *part, PackedNote *notes, uint32_t hq,
                               float scale) {
    brasa_ctx *ctx = cmd->ctx;
    PackedMaps maps;
    const uint64_t dims[3] = {D, v.hkv, (uint64_t)v.num_pages * PAGE}, strides[2] = {256, (uint64_t)v.hkv * 256};
    const uint32_t box[3] = {64, 1, PAGE};
    BRASA_TRY(brasa_tmap_bf16(ctx, &maps.k, 3, kpool, dims, strides, box));  // (16-bit values are copied whatever they are)
    BRASA_TRY(brasa_tmap_bf16(ctx, &maps.v, 3, vpool, dims, strides, box));
    const PackedTcParams p{packed_line(v, hq / v.hkv, ROWS, 7, 2, 2, 4, PACKED_TC_MIN_ROWS, UINT32_MAX), q, vpool, (__half *)o, part, notes, hq, scale, ctx->status};
    const size_t smem = (2 + SLOTS) * TILE_BYTES + SOFTMAX_WARPS * 2048;
    BRASA_TRY(brasa_smem_optin(ctx, (const void *)attn_packed_tc_kernel, smem));
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, attn_packed_tc_kernel, dim3(ctx->sm_count), dim3(THREADS), smem, maps, p));
    return brasa_post_launch(cmd, "attn_packed_tc");
}
