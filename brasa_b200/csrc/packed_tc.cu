// Attention of a packed run's sequences of many rows on the 5th-generation tensor cores (F16 precision, f16 caches), over pages.
//
// An item is 256 rows of one sequence against one key head, in two tiles of 128; a row is a token and a head of the group, so that short
// prompts of grouped heads fill their tiles and all heads of a group share K and V. Per tile of 128 keys and row tile there are two products of
// 128^3: S = Q K^T into tensor memory, O += P V with P read out of tensor memory, over the columns that S had. Two threads hold a row, 64 scores
// each: warps 0-7 tile A, 8-15 tile B; warp 16 issues the products, warp 17 the copies. The order on the tensor core is P V of A, S of
// A's next keys, P V of B, S of B's next, so that one tile's products run while the other's probabilities are formed.
// K and V tiles are eight pages each, two boxes of 16 positions x 64 dims a page (cp.async.bulk.tensor, 128-byte swizzle), through a ring of five
// 32 KB slots. Rows of the cache behind the item's last position may hold anything: such scores are replaced before they count, and V's rows,
// which enter P V with a weight of zero, are written as zeros by the copying warp instead of copied.
// What bounds it: the tensor core, 2 048 cycles per tile of keys, and as many cycles of exponentials (16 a clock).
#include <math.h>

#include "packed_tc.h"
#include "tc_device.cuh"

using namespace brasa_dev;

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE, D = 128, WAIT_LIMIT = 1u << 22, TILE_BYTES = 128 * 128 * 2, SLOTS = 5, ROWS = PACKED_TC_ROWS;
constexpr uint32_t SOFTMAX_THREADS = 512, THREADS = SOFTMAX_THREADS + 64;

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
    __shared__ uint64_t full[SLOTS], freed[SLOTS], s_ready[2], p_ready[2], o_done[2];
    __shared__ uint32_t tmem_base_s, abort_s;
    __shared__ float pair[2][2][128];  // [tile][half of the keys][row]: largest score
    __shared__ PackedPieces pieces;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.l.group, hkv = p.l.v.hkv;

    if (tid == 0) {
        for (uint32_t i = 0; i < SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&freed[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_ready[i], 1);
            mbar_init(&p_ready[i], 8);  // one arrival per softmax warp
            mbar_init(&o_done[i], 1);
        }
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {  // tensor memory: S, then P, of A in [0, 128), of B in [128, 256); O of A in [256, 384), of B in [384, 512)
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

    if (smem_u32(smem) & 1023) {  // (the swizzle counts from there)
        if (tid == 0) atomicExch(p.status, 8u);
        abort_s = 1;
    }
    const bool work = line_cut<256>(p.l, pieces) && !abort_s;
    PackedItem item = pieces.at[0];
    const uint64_t end_first = pieces.at[1].first;
    const uint32_t end_j = pieces.at[1].j;
    if (work && item.j == item.tiles) line_next(p.l, item);
    PackedNote note{};
    uint32_t loads = 0, done_tiles[2] = {0, 0}, segs[2] = {0, 0};  // of this block so far: tiles copied (K and V apart), key tiles and items by row tile
#pragma unroll 1
    while (work && (item.first < end_first || (item.first == end_first && item.j < end_j))) {
        const uint32_t j0 = item.j, j1 = item.first == end_first ? end_j : item.tiles, len = j1 - j0;
        const uint32_t row0 = item.part * ROWS, rows = min(ROWS, item.rows - row0), nx = rows > 128 ? 2 : 1, nkeys = line_keys(p.l, item, item.part);
        const int32_t *table = p.l.v.table + (size_t)item.seq * p.l.v.max_pages;
        auto page_at = [&](uint32_t j, uint32_t i) -> int32_t {  // page i of key tile j, -1 where nothing is seen
            const int32_t page = j < j1 && 128 * j + 16 * i < nkeys ? table[8 * j + i] : -1;
            return (uint32_t)page < p.l.v.num_pages ? page : -1;
        };
        // ---- copies: lanes 2 i and 2 i + 1 of warp 17 take the halves of page i ----
        uint32_t n = loads;
        const uint32_t n_end = loads + 2 * len;
        int32_t pg = -1;
        auto load = [&]() -> bool {  // (the whole warp) K and V of a tile in turn
            const uint32_t s = n % SLOTS, j = j0 + (n - loads) / 2, half = lane & 1, i = (lane >> 1) & 7;
            const bool is_v = (n - loads) & 1;
            if (n >= SLOTS && !__all_sync(0xffffffffu, wait(&freed[s], ((n / SLOTS) - 1) & 1))) return false;
            uint8_t *slot = ring + (size_t)s * TILE_BYTES;
            const uint32_t left = nkeys - min(nkeys, 128 * j + 16 * i);  // of the page's positions, those that are seen
            const bool whole_page = pg >= 0 && (!is_v || left >= 16);
            if (is_v && __any_sync(0xffffffffu, !whole_page)) {  // rows that must be zeros, beside those of a page that is seen in part
                if (!whole_page && lane < 16) {
                    for (uint32_t r = 0; r < 16; ++r) {
                        const bool seen = pg >= 0 && r < left;
                        const uint4 *src = reinterpret_cast<const uint4 *>(p.vpool + (((size_t)max(pg, 0) * PAGE + r) * hkv + item.kh) * 256 + 128 * half);
                        for (uint32_t c = 0; c < 8; ++c)
                            *reinterpret_cast<uint4 *>(slot + tile_piece(16 * i + r, 64 * half + 8 * c)) = seen ? src[c] : make_uint4(0, 0, 0, 0);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            const uint32_t copies = __popc(__ballot_sync(0xffffffffu, whole_page && lane < 16));
            if (lane == 0) mbar_expect_tx(&full[s], copies * 2048);
            __syncwarp();
            if (whole_page && lane < 16) tma_load_3d(slot + half * 16384 + i * 2048, is_v ? &maps.v : &maps.k, (int)(half * 64), (int)item.kh, pg * (int)PAGE, &full[s]);
            if (is_v) pg = page_at(j + 1, i);
            ++n;
            return true;
        };
        if (warp == 17) {  // (every slot is free here: the item before has used them all up)
            pg = page_at(j0, (lane >> 1) & 7);
            for (uint32_t k = 0; k < SLOTS && n < n_end && load(); ++k) {}
        } else if (warp < 16) {
            // Q tiles: scale, round to f16, swizzled K-major; rows past the last are zeros
#pragma unroll 1
            for (uint32_t i0 = tid; i0 < nx * 128 * 16; i0 += 4 * SOFTMAX_THREADS) {
                float4 v[4][2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t i = i0 + SOFTMAX_THREADS * k, r = row0 + (i >> 4);
                    v[k][0] = v[k][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (i < nx * 128 * 16 && r < item.rows) {
                        const float4 *src = reinterpret_cast<const float4 *>(p.q + ((size_t)(item.t0 + r / G) * p.hq + item.kh * G + r % G) * D + (i & 15) * 8);
                        v[k][0] = src[0];
                        v[k][1] = src[1];
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t i = i0 + SOFTMAX_THREADS * k;
                    const float4 a = v[k][0], b = v[k][1];
                    const __half2 h0 = __floats2half2_rn(a.x * p.scale, a.y * p.scale), h1 = __floats2half2_rn(a.z * p.scale, a.w * p.scale);
                    const __half2 h2 = __floats2half2_rn(b.x * p.scale, b.y * p.scale), h3 = __floats2half2_rn(b.z * p.scale, b.w * p.scale);
                    if (i < nx * 128 * 16)
                        *reinterpret_cast<uint4 *>(smem + (i >> 11) * TILE_BYTES + tile_piece((i >> 4) & 127, (i & 15) * 8)) =
                            make_uint4(*reinterpret_cast<const uint32_t *>(&h0), *reinterpret_cast<const uint32_t *>(&h1), *reinterpret_cast<const uint32_t *>(&h2),
                                       *reinterpret_cast<const uint32_t *>(&h3));
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

        if (warp == 17) {  // ---- the other copies ----
            while (n < n_end && load()) {}
            if (*abort_flag && lane == 0) {  // leaving early: let the copies in flight land before the block's shared memory is handed on
                for (uint32_t k = n > SLOTS ? n - SLOTS : 0; k < n; ++k)
                    for (uint32_t it = 0; it < WAIT_LIMIT && !tc_mbar_try(&full[k % SLOTS], (k / SLOTS) & 1); ++it) {}
            }
        } else if (warp == 16) {  // ---- products: the warp waits, one lane issues ----
            const uint32_t idesc_s = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24), idesc_o = idesc_s | (1u << 16);  // f16 operands; V is MN-major
            auto all_wait = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
            auto landed = [&](uint32_t m) { return all_wait(&full[m % SLOTS], (m / SLOTS) & 1); };
            auto slot = [&](uint32_t m) { return smem_u32(ring + (size_t)(m % SLOTS) * TILE_BYTES); };
            bool ok = true;
            for (uint32_t j = 0; j <= len && ok; ++j) {
                for (uint32_t x = 0; x < nx && ok; ++x) {
                    if (j > 0) {  // O += P V of the tile before
                        const uint32_t m = loads + 2 * (j - 1) + 1, o = tmem + 256 + 128 * x, ph = tmem + 128 * x;
                        ok = all_wait(&p_ready[x], (done_tiles[x] + j - 1) & 1) && landed(m);
                        if (!ok) break;
                        if (tc_elect_one()) {
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint32_t v = slot(m);
#pragma unroll
                            for (uint32_t ks = 0; ks < 8; ++ks)  // 16 keys: 8 columns of P; each thread's 64 keys begin at its own scores
                                tc_mma_ta(o, ph + 64 * (ks >> 2) + 8 * (ks & 3), tc_desc_mnmajor(v + ks * 2048), idesc_o, (j > 1 || ks > 0) ? 1u : 0u);
                            if (x + 1 == nx) tc_commit(&freed[m % SLOTS]);
                            if (j == len) tc_commit(&o_done[x]);
                        }
                        __syncwarp();
                    }
                    if (j < len) {  // S = Q K^T of this tile, over the columns of the P just read
                        const uint32_t m = loads + 2 * j, q = smem_u32(smem + x * TILE_BYTES);
                        if (!(ok = landed(m))) break;
                        if (tc_elect_one()) {
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint32_t k = slot(m);
#pragma unroll
                            for (uint32_t ks = 0; ks < 8; ++ks) {
                                const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
                                tc_mma(tmem + 128 * x, tc_desc_kmajor(q + off), tc_desc_kmajor(k + off), idesc_s, ks > 0 ? 1u : 0u);
                            }
                            if (x + 1 == nx) tc_commit(&freed[m % SLOTS]);
                            tc_commit(&s_ready[x]);
                        }
                        __syncwarp();
                    }
                }
            }
        } else if ((warp >> 3) < nx) {  // ---- softmax: two threads per row, 64 keys of every tile each ----
            constexpr float LOG2E = 1.4426950408889634f, SLACK = 5.545177444f;  // 8 ln 2
            const uint32_t x = warp >> 3, h = (warp >> 2) & 1, row = (warp & 3) * 32 + lane, r = row0 + 128 * x + row;
            const bool live = r < item.rows;
            const uint32_t seen_all = live ? item.past + r / G + 1 : 0;
            const uint32_t nfree = (item.past + (row0 + 128 * x) / G + 1) / 128;  // tiles [0, nfree) lie wholly at or below every row's own position
            const uint32_t trow = ((warp & 3) * 32u) << 16, ts = tmem + 128 * x + 64 * h + trow, to = tmem + 256 + 128 * x + 64 * h + trow;
            const uint32_t both = 1 + 4 * x + (warp & 3);  // named barrier of the two warps that hold these rows
            float m = -INFINITY, mneg = 0.0f, l0 = 0.0f, l1 = 0.0f;
            bool ok = true;
            int32_t mine = page_at(j0, 4 * h + (lane & 3));  // the four pages of this warp's keys
            for (uint32_t j = j0; j < j1; ++j) {
                const uint32_t there = __ballot_sync(0xffffffffu, mine >= 0) & 15;
                mine = page_at(j + 1, 4 * h + (lane & 3));
                ok = wait(&s_ready[x], (done_tiles[x] + j - j0) & 1);  // S of this tile, and with it every product issued before: P V of the tile before
                ok = __all_sync(0xffffffffu, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t v[2][32];
                tmem_ld32(ts, v[0]);
                tmem_ld32(ts + 32, v[1]);
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
                tmax = fmaxf(pair[x][0][row], pair[x][1][row]);
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
                }
                if (__any_sync(0xffffffffu, move)) {  // what O holds for the row was accumulated against the old reference
#pragma unroll 1
                    for (uint32_t c = 0; c < 64; c += 32) {
                        uint32_t o[32];
                        tc_ld32(to + c, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * rescale);
                        tc_st32(to + c, o);
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) tc_mbar_arrive(&p_ready[x]);
            }
            // ---- output: O / l, rounded to f16; a part of the item's keys: O, m and l as they are ----
            ok = ok && wait(&o_done[x], segs[x] & 1);
            ok = __all_sync(0xffffffffu, ok);
            float *sums = reinterpret_cast<float *>(smem + x * TILE_BYTES);  // [half][row], over the Q tile: its products are done
            if (ok) sums[h * 128 + row] = l0 + l1;
            ok = tc_pair_agree(both, ok);
            if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float l = sums[row] + sums[128 + row];
                if (len < item.tiles) {
                    float *dst = p.part + (size_t)(2 * blockIdx.x + (j0 == 0)) * packed_part_floats(ROWS);
                    if (h == 0 && live) {
                        dst[ROWS * D + 128 * x + row] = m * LOG2E;
                        dst[ROWS * D + ROWS + 128 * x + row] = l;
                    }
#pragma unroll 1
                    for (uint32_t c = 0; c < 2; ++c) {
                        uint32_t o[32];
                        tc_ld32(to + 32 * c, o);
#pragma unroll
                        for (int g = 0; g < 8; ++g)
                            if (live) reinterpret_cast<uint4 *>(dst + (size_t)(128 * x + row) * D)[16 * h + 8 * c + g] = make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
                    }
                } else {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    uint4 *dst = reinterpret_cast<uint4 *>(p.o + ((size_t)(item.t0 + (live ? r / G : 0)) * p.hq + item.kh * G + (live ? r % G : 0)) * D + 64 * h);
#pragma unroll 1
                    for (uint32_t c = 0; c < 2; ++c) {
                        uint32_t o[32], packed[16];
                        tc_ld32(to + 32 * c, o);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const __half2 hh = __floats2half2_rn(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                            packed[i >> 1] = *reinterpret_cast<const uint32_t *>(&hh);
                        }
#pragma unroll
                        for (int g = 0; g < 4; ++g)
                            if (live) dst[4 * c + g] = make_uint4(packed[4 * g], packed[4 * g + 1], packed[4 * g + 2], packed[4 * g + 3]);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            }
        }
        loads += 2 * len;
        for (uint32_t x = 0; x < nx; ++x) {
            done_tiles[x] += len;
            ++segs[x];
        }
        if (len < item.tiles && j0 == 0) note = PackedNote{1, note.closes, item.t0 + row0 / G, row0 % G, rows, item.kh};
        if (j0 > 0 && j1 == item.tiles) note.closes = 1;
        const bool more = j1 == item.tiles && line_next(p.l, item);
        if (__syncthreads_or(*abort_flag) || !more) break;  // Q, the row sums and O are free again
    }
    if (tid == 0) p.notes[blockIdx.x] = note;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 16) {
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
    const PackedTcParams p{{v, hq / v.hkv, ROWS, 128, 2, 3, 6, PACKED_TC_MIN_ROWS, UINT32_MAX}, q, vpool, (__half *)o, part, notes, hq, scale, ctx->status};
    const size_t smem = (2 + SLOTS) * TILE_BYTES;
    BRASA_TRY(brasa_smem_optin(ctx, (const void *)attn_packed_tc_kernel, smem));
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, attn_packed_tc_kernel, dim3(ctx->sm_count), dim3(THREADS), smem, maps, p));
    return brasa_post_launch(cmd, "attn_packed_tc");
}
