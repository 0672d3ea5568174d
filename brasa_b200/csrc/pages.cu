// Pages of a cache handed from rows to rows: brasa_k_pages_reassign (fork, reorder, roll back, free, reserve, with a copy of every last page
// that two rows would write into) and brasa_k_pages_compact. Each is a plan, made by one block, and a copy of whole pages over all layers
// by a dependent kernel that reads how many there are. The plan is integer work on a few thousand words, bound by the latency of its steps;
// flags of pages are bits in shared memory, and every rank (of free pages, of rows, of copies) is a prefix sum, so that the outcome does not
// depend on the order in which threads arrive. The copies are bound by memory: a page read once and written once per layer, K and V.
// 64 rows after a verified step 11 us, nearly all of it the two launches and the plan's steps; 48 rows of 8 prompts (36 layers, 8 bit) with 35 pages copied 22 us, 4 TB/s;
// 24 layers moved to the front of their pool 89 us, 4.6 TB/s (one piece a thread at a time: 25 us for the 22).
#include "brasa_internal.h"

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE, THREADS = 1024, WARPS = THREADS / 32, MAX_PAGES = 1u << 19, MAX_ROWS = 65536;

struct PagePlan {
    const int32_t *table;
    const uint32_t *lens, *pinned;
    uint32_t rows, max_pages, num_pages;
    int32_t *table_out;
    uint32_t *result;
    // workspace
    uint32_t *owner, *free_list;  // [num_pages]: first row that ends in a page; free pages in order
    uint32_t *first;              // [rows]: how many pages are handed out before the row's, top bit: its last page is copied
    uint32_t *copies;             // [0] how many, then (from, to) pairs [max(rows, num_pages)]
};

__device__ __forceinline__ bool bit(const uint32_t *bits, uint32_t i) { return bits[i >> 5] >> (i & 31) & 1; }
__device__ __forceinline__ void set_bit(uint32_t *bits, uint32_t i) { atomicOr(&bits[i >> 5], 1u << (i & 31)); }

// The sum of v over the block's threads before this one; the whole in `total`.
__device__ uint32_t block_scan(uint32_t v, uint32_t *sums, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t upto = v;
    for (uint32_t x = 1; x < 32; x <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += o;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = sums[lane];
        for (uint32_t x = 1; x < 32; x <<= 1) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, s, x);
            if (lane >= x) s += o;
        }
        sums[lane] = s;
    }
    __syncthreads();
    total = sums[WARPS - 1];
    return upto - v + (warp ? sums[warp - 1] : 0);
}

struct NewRow {
    uint32_t source, keep, have, want, whole;  // old row; positions kept; pages that hold them; pages in all; full ones among the kept
};
struct ReassignArgs {
    PagePlan p;
    const int32_t *source;
    const uint32_t *keep, *accepted, *starts, *room;
    uint32_t *lens_out;
};
__device__ __forceinline__ NewRow new_row(const ReassignArgs &a, uint32_t r) {
    NewRow n;
    const int32_t s = a.source[r];
    const bool there = (uint32_t)s < a.p.rows;
    const uint64_t most = (uint64_t)a.p.max_pages * PAGE;
    n.source = there ? (uint32_t)s : 0u;
    uint64_t holds = 0;
    if (there) holds = (uint64_t)a.p.lens[s] + (a.accepted && (!a.starts || a.starts[s + 1] > a.starts[s]) ? (uint64_t)a.accepted[s] + 1 : 0);
    if (a.keep) holds = min(holds, (uint64_t)a.keep[r]);
    n.keep = (uint32_t)min(holds, most);
    n.have = (n.keep + PAGE - 1) / PAGE;
    n.want = (uint32_t)((min((uint64_t)n.keep + a.room[r], most) + PAGE - 1) / PAGE);
    n.whole = n.keep / PAGE;
    return n;
}
__device__ __forceinline__ int32_t valid_page(const PagePlan &p, int32_t page) { return (uint32_t)page < p.num_pages ? page : -1; }

// Bits of pinned pages; owner as no row's.
__device__ void plan_begin(const PagePlan &p, uint32_t *used, uint32_t *shared, uint32_t words) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t i = threadIdx.x; i < words * 32; i += THREADS) {  // (words is a multiple of 32: whole warps go round)
        const uint32_t b = __ballot_sync(0xffffffffu, i < p.num_pages && p.pinned && p.pinned[i] != 0);
        if (lane == 0) {
            used[i >> 5] = b;
            if (shared) shared[i >> 5] = b;
        }
        if (i < p.num_pages && shared) p.owner[i] = UINT32_MAX;
    }
    __syncthreads();
}

// Free pages in order, as far as `most`; returns how many there are in all.
__device__ uint32_t plan_free(const PagePlan &p, const uint32_t *used, uint32_t words, uint32_t most, uint32_t *sums) {
    const uint32_t each = (words + THREADS - 1) / THREADS, w0 = min(threadIdx.x * each, words), w1 = min(w0 + each, words);
    uint32_t mine = 0, total;
    auto free_bits = [&](uint32_t w) {
        const uint32_t left = p.num_pages - min(p.num_pages, w * 32);
        return ~used[w] & (left >= 32 ? 0xffffffffu : (1u << left) - 1u);
    };
    for (uint32_t w = w0; w < w1; ++w) mine += __popc(free_bits(w));
    uint32_t at = block_scan(mine, sums, total);
    for (uint32_t w = w0; w < w1 && at < most; ++w)
        for (uint32_t b = free_bits(w); b && at < most; b &= b - 1) p.free_list[at++] = w * 32 + __ffs(b) - 1;
    __syncthreads();
    return total;
}

__global__ void __launch_bounds__(THREADS) pages_reassign_kernel(ReassignArgs a, uint32_t words) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched as a programmatic dependent: see brasa_launch_dependent)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint32_t bits[];
    __shared__ uint32_t sums[32];
    const PagePlan &p = a.p;
    uint32_t *used = bits, *shared = bits + words;  // held by a new row or pinned; held whole or pinned
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    plan_begin(p, used, shared, words);
    // ---- what the new rows hold ----
    for (uint32_t r = warp; r < p.rows; r += WARPS) {
        const NewRow n = new_row(a, r);
        const int32_t *old = p.table + (size_t)n.source * p.max_pages;
        for (uint32_t i = lane; i < n.have; i += 32) {
            const int32_t page = valid_page(p, old[i]);
            if (page < 0) continue;
            set_bit(used, page);
            if (i < n.whole) set_bit(shared, page);
            else atomicMin(&p.owner[page], r);
        }
    }
    __syncthreads();
    // ---- what each row needs, and its place in the line ----
    uint32_t need_all = 0, copies_all = 0;
    for (uint32_t r0 = 0; r0 < p.rows; r0 += THREADS) {
        const uint32_t r = r0 + tid;
        uint32_t need = 0, copy = 0;
        if (r < p.rows) {
            const NewRow n = new_row(a, r);
            if (n.have > n.whole) {
                const int32_t tail = valid_page(p, p.table[(size_t)n.source * p.max_pages + n.whole]);
                copy = tail >= 0 && (bit(shared, tail) || p.owner[tail] != r);
            }
            need = copy + n.want - n.have;
        }
        uint32_t total, copies;
        const uint32_t at = need_all + block_scan(need, sums, total), c = block_scan(copy, sums, copies);
        if (r < p.rows) p.first[r] = at;
        if (copy) {
            const NewRow n = new_row(a, r);
            p.copies[1 + 2 * (size_t)(copies_all + c)] = (uint32_t)p.table[(size_t)n.source * p.max_pages + n.whole];
            p.copies[2 + 2 * (size_t)(copies_all + c)] = at;  // (a place in the free list until that is made)
            p.first[r] = at | 1u << 31;
        }
        need_all += total;
        copies_all += copies;
    }
    __syncthreads();
    const uint32_t free_all = plan_free(p, used, words, need_all, sums);
    const bool short_of = need_all > free_all;
    if (!short_of)
        for (uint32_t i = tid; i < copies_all; i += THREADS) p.copies[2 + 2 * (size_t)i] = p.free_list[p.copies[2 + 2 * (size_t)i]];
    // ---- the new table ----
    uint32_t kept_all = 0;
    if (short_of) {  // as it was; in use is what it names
        __syncthreads();
        plan_begin(p, used, nullptr, words);
    }
    for (uint32_t r = warp; r < p.rows; r += WARPS) {
        const NewRow n = new_row(a, r);
        const uint32_t at = p.first[r] & ~(1u << 31), copy = p.first[r] >> 31;
        const int32_t *old = p.table + (size_t)(short_of ? r : n.source) * p.max_pages;
        for (uint32_t i = lane; i < p.max_pages; i += 32) {
            int32_t page = -1;
            if (short_of) {
                page = valid_page(p, old[i]);
                if (page >= 0) set_bit(used, page);
            } else if (copy && i == n.whole) page = (int32_t)p.free_list[at];
            else if (i < n.have) page = valid_page(p, old[i]);
            else if (i < n.want) page = (int32_t)p.free_list[at + copy + i - n.have];
            p.table_out[(size_t)r * p.max_pages + i] = page;
        }
        if (lane == 0) a.lens_out[r] = short_of ? p.lens[r] : n.keep;
    }
    __syncthreads();
    for (uint32_t w = tid; w < words; w += THREADS) kept_all += __popc(used[w]);
    uint32_t in_use;
    block_scan(kept_all, sums, in_use);
    if (tid == 0) {
        if (!short_of) in_use += need_all;
        p.copies[0] = short_of ? 0 : copies_all;
        p.result[0] = in_use;
        p.result[1] = short_of ? 0 : copies_all;
        p.result[2] = p.num_pages - in_use;
        p.result[3] = short_of ? need_all - free_all : 0;
    }
}

__global__ void __launch_bounds__(THREADS) pages_compact_kernel(PagePlan p, uint32_t *moved, uint32_t words) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint32_t bits[];
    __shared__ uint32_t sums[32], end_s;
    uint32_t *used = bits;
    const uint32_t tid = threadIdx.x;
    plan_begin(p, used, nullptr, words);
    const size_t entries = (size_t)p.rows * p.max_pages;
    for (size_t i = tid; i < entries; i += THREADS) {
        const int32_t page = valid_page(p, p.table[i]);
        if (page >= 0 && !bit(used, page)) set_bit(used, page);
    }
    if (tid == 0) end_s = 0;
    __syncthreads();
    // ---- the i-th free page from the front and the i-th page that may move from the back: a pair while the free one is the lower ----
    const uint32_t holes = plan_free(p, used, words, p.num_pages, sums);
    const uint32_t each = (words + THREADS - 1) / THREADS, w0 = min(tid * each, words), w1 = min(w0 + each, words);
    auto movable = [&](uint32_t w) {
        uint32_t b = used[w];
        if (p.pinned)
            for (uint32_t c = b; c; c &= c - 1) {
                const uint32_t i = w * 32 + __ffs(c) - 1;
                if (p.pinned[i]) b &= ~(1u << (i & 31));
            }
        return b;
    };
    uint32_t mine = 0, used_mine = 0, movers, in_use;
    for (uint32_t w = w0; w < w1; ++w) {
        mine += __popc(movable(w));
        used_mine += __popc(used[w]);
    }
    uint32_t at = block_scan(mine, sums, movers);
    block_scan(used_mine, sums, in_use);
    uint32_t pairs = 0;
    for (uint32_t w = w0; w < w1; ++w) {
        uint32_t can = movable(w);
        for (uint32_t b = 0; b < 32 && w * 32 + b < p.num_pages; ++b) {
            const uint32_t page = w * 32 + b;
            int32_t to = bit(used, page) ? (int32_t)page : -1;
            if (can >> b & 1) {
                const uint32_t i = movers - 1 - at++;  // from the back
                if (i < holes && p.free_list[i] < page) {
                    to = (int32_t)p.free_list[i];
                    p.copies[1 + 2 * (size_t)i] = page;
                    p.copies[2 + 2 * (size_t)i] = (uint32_t)to;
                    ++pairs;
                }
            }
            moved[page] = to;
            if (to >= 0) atomicMax(&end_s, (uint32_t)to + 1);
        }
    }
    uint32_t all;
    block_scan(pairs, sums, all);  // (its barriers also publish `moved`)
    if (tid == 0) {
        p.copies[0] = all;
        p.result[0] = in_use;
        p.result[1] = all;
        p.result[2] = end_s;
        p.result[3] = 0;
    }
    for (size_t i = tid; i < entries; i += THREADS) {
        const int32_t page = valid_page(p, p.table[i]);
        p.table_out[i] = page >= 0 ? moved[page] : -1;
    }
}

// Pages in 16-byte pieces, COPY_PIECES to a block's turn (four a thread, asked for together); an item is one such part of one page of one layer's K or V.
constexpr uint32_t COPY_THREADS = 256, COPY_PIECES = 4 * COPY_THREADS;
__global__ void __launch_bounds__(COPY_THREADS) pages_copy_kernel(uint8_t *kpool, uint8_t *vpool, const uint32_t *copies, uint32_t pieces, uint32_t layers, uint32_t num_pages) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t parts = (pieces + COPY_PIECES - 1) / COPY_PIECES, planes = 2 * layers, tid = threadIdx.x;
    const uint64_t items = (uint64_t)copies[0] * planes * parts;
    for (uint64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const uint32_t part = (uint32_t)(it % parts), plane = (uint32_t)(it / parts % planes);
        const uint64_t c = it / parts / planes;
        uint4 *pool = reinterpret_cast<uint4 *>(plane & 1 ? vpool : kpool) + (uint64_t)(plane >> 1) * num_pages * pieces;
        const uint4 *from = pool + (uint64_t)copies[1 + 2 * c] * pieces;
        uint4 *to = pool + (uint64_t)copies[2 + 2 * c] * pieces;
        uint4 v[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t i = part * COPY_PIECES + u * COPY_THREADS + tid;
            if (i < pieces) v[u] = from[i];
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t i = part * COPY_PIECES + u * COPY_THREADS + tid;
            if (i < pieces) to[i] = v[u];
        }
    }
}

int32_t check_pool(brasa_ctx *ctx, const char *who, const brasa_page_pool &g) {
    BRASA_REQUIRE(ctx, g.kv >= BRASA_KV_F32 && g.kv <= BRASA_KV_Q8_0, "%s: unknown KV type %d", who, g.kv);
    BRASA_REQUIRE(ctx, g.rows >= 1 && g.max_pages >= 1 && g.num_pages >= 1 && g.layers >= 1 && g.hkv >= 1, "%s: empty pool or table", who);
    BRASA_REQUIRE(ctx, g.rows <= MAX_ROWS && g.num_pages <= MAX_PAGES && g.max_pages <= MAX_PAGES && g.layers <= 65536 && g.hkv <= 65536,
                  "%s: more than %u rows, %u pages, or 65 536 layers or heads", who, MAX_ROWS, MAX_PAGES);
    BRASA_REQUIRE(ctx, (uint64_t)g.rows * g.max_pages <= 1ull << 30, "%s: a table of more than 2^30 entries", who);
    const uint64_t page = brasa_kv_bytes(g.kv, (uint64_t)PAGE * g.hkv * 128), layer = page * g.num_pages;
    BRASA_REQUIRE(ctx, layer <= UINT64_MAX / g.layers && arg_fits(g.kpool, layer * g.layers) && arg_fits(g.vpool, layer * g.layers), "%s: the pools are smaller than num_pages pages of all layers", who);
    BRASA_REQUIRE(ctx, arg_fits(g.table, (uint64_t)g.rows * g.max_pages * 4) && arg_fits(g.lens, (uint64_t)g.rows * 4) &&
                  (!g.pinned.buf || arg_fits(g.pinned, (uint64_t)g.num_pages * 4)), "%s: table, lens or pinned too small", who);
    BRASA_REQUIRE(ctx, g.kpool.offset % 16 == 0 && g.vpool.offset % 16 == 0 && g.table.offset % 4 == 0 && g.lens.offset % 4 == 0 && g.pinned.offset % 4 == 0, "%s: misaligned", who);
    return BRASA_OK;
}
uint64_t pool_bytes(const brasa_page_pool &g) { return brasa_kv_bytes(g.kv, (uint64_t)PAGE * g.hkv * 128) * g.num_pages * g.layers; }  // (of K or V, behind check_pool)
// The plan's arrays in the context's workspace.
int32_t plan_of(brasa_ctx *ctx, const brasa_page_pool &g, brasa_arg table_out, brasa_arg result, PagePlan *p) {
    const size_t pairs = std::max(g.rows, g.num_pages), words = 2 * (size_t)g.num_pages + g.rows + 4 + 2 * pairs;
    BRASA_TRY(brasa_workspace(ctx, (void **)&ctx->page_work, &ctx->page_work_bytes, words * 4));
    uint32_t *w = (uint32_t *)ctx->page_work;
    *p = PagePlan{(const int32_t *)arg_ptr(g.table), (const uint32_t *)arg_ptr(g.lens), (const uint32_t *)arg_ptr(g.pinned), g.rows, g.max_pages, g.num_pages,
                  (int32_t *)arg_ptr(table_out), (uint32_t *)arg_ptr(result), w, w + g.num_pages, w + 2 * (size_t)g.num_pages, w + 2 * (size_t)g.num_pages + g.rows};
    return BRASA_OK;
}
uint32_t flag_words(uint32_t num_pages) { return (num_pages + 1023) / 1024 * 32; }

int32_t copy_pages(brasa_cmd *cmd, const brasa_page_pool &g, const PagePlan &p) {
    brasa_ctx *ctx = cmd->ctx;
    const uint32_t pieces = (uint32_t)(brasa_kv_bytes(g.kv, (uint64_t)PAGE * g.hkv * 128) / 16);
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, pages_copy_kernel, dim3(ctx->sm_count * 8), dim3(COPY_THREADS), 0, arg_ptr(g.kpool), arg_ptr(g.vpool), (const uint32_t *)p.copies, pieces,
                                           g.layers, g.num_pages));
    return brasa_post_launch(cmd, "pages_copy");
}

}  // namespace

extern "C" {

int32_t brasa_k_pages_reassign(brasa_cmd *cmd, brasa_page_pool g, brasa_arg source, brasa_arg keep, brasa_arg accepted, brasa_arg starts, brasa_arg room,
                               brasa_arg table_out, brasa_arg lens_out, brasa_arg result) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    BRASA_TRY(check_pool(ctx, "pages_reassign", g));
    const uint64_t nt = (uint64_t)g.rows * g.max_pages * 4, nr = (uint64_t)g.rows * 4;
    BRASA_REQUIRE(ctx, arg_fits(source, nr) && (!keep.buf || arg_fits(keep, nr)) && (!accepted.buf || arg_fits(accepted, nr)) && (!starts.buf || arg_fits(starts, nr + 4)) && arg_fits(room, nr),
                  "pages_reassign: source, keep, accepted, starts or room too small");
    BRASA_REQUIRE(ctx, accepted.buf || !starts.buf, "pages_reassign: starts without accepted");
    BRASA_REQUIRE(ctx, arg_fits(table_out, nt) && arg_fits(lens_out, nr) && arg_fits(result, 16), "pages_reassign: table_out, lens_out or result too small");
    for (const brasa_arg *a : {&source, &keep, &accepted, &starts, &room, &table_out, &lens_out, &result}) BRASA_REQUIRE(ctx, a->offset % 4 == 0, "pages_reassign: misaligned buffer");
    const uint64_t np = (uint64_t)g.num_pages * 4, pool = pool_bytes(g);
    const brasa_range table{table_out, nt}, lens{lens_out, nr}, counts{result, 16}, k{g.kpool, pool}, v{g.vpool, pool};
    const bool over = any_overlap({table, lens, counts, k, v}, {{g.table, nt}, {g.lens, nr}, {source, nr}, {keep, nr}, {accepted, nr}, {starts, nr + 4}, {room, nr}, {g.pinned, np}}) ||
                      any_overlap({table, lens, counts}, {k, v}) || any_overlap({table}, {lens, counts}) || any_overlap({lens}, {counts});
    BRASA_REQUIRE(ctx, !over, "pages_reassign: table_out, lens_out, result and the pools must overlap neither one another nor what is read");
    ReassignArgs a;
    BRASA_TRY(plan_of(ctx, g, table_out, result, &a.p));
    a.source = (const int32_t *)arg_ptr(source);
    a.keep = (const uint32_t *)arg_ptr(keep);
    a.accepted = (const uint32_t *)arg_ptr(accepted);
    a.starts = (const uint32_t *)arg_ptr(starts);
    a.room = (const uint32_t *)arg_ptr(room);
    a.lens_out = (uint32_t *)arg_ptr(lens_out);
    const uint32_t words = flag_words(g.num_pages);
    BRASA_TRY(brasa_smem_optin(ctx, (const void *)pages_reassign_kernel, 2 * words * 4));
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, pages_reassign_kernel, dim3(1), dim3(THREADS), 2 * words * 4, a, words));
    BRASA_TRY(brasa_post_launch(cmd, "pages_reassign"));
    return copy_pages(cmd, g, a.p);
}

int32_t brasa_k_pages_compact(brasa_cmd *cmd, brasa_page_pool g, brasa_arg table_out, brasa_arg moved, brasa_arg result) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    BRASA_TRY(check_pool(ctx, "pages_compact", g));
    const uint64_t nt = (uint64_t)g.rows * g.max_pages * 4, np = (uint64_t)g.num_pages * 4;
    BRASA_REQUIRE(ctx, arg_fits(table_out, nt) && arg_fits(moved, np) && arg_fits(result, 16), "pages_compact: table_out, moved or result too small");
    for (const brasa_arg *a : {&table_out, &moved, &result}) BRASA_REQUIRE(ctx, a->offset % 4 == 0, "pages_compact: misaligned buffer");
    const bool in_place = table_out.buf == g.table.buf && table_out.offset == g.table.offset;
    const uint64_t pool = pool_bytes(g);
    const brasa_range table{table_out, nt}, where{moved, np}, counts{result, 16}, k{g.kpool, pool}, v{g.vpool, pool};
    const bool over = (!in_place && arg_overlap(table_out, nt, g.table, nt)) || any_overlap({where, counts, k, v}, {{g.table, nt}, {g.pinned, np}}) ||
                      any_overlap({table}, {{g.pinned, np}, where, counts, k, v}) || any_overlap({where, counts}, {k, v}) || any_overlap({where}, {counts});
    BRASA_REQUIRE(ctx, !over, "pages_compact: outputs and the pools overlap one another or what is read");
    PagePlan p;
    BRASA_TRY(plan_of(ctx, g, table_out, result, &p));
    const uint32_t words = flag_words(g.num_pages);
    BRASA_TRY(brasa_smem_optin(ctx, (const void *)pages_compact_kernel, words * 4));
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, pages_compact_kernel, dim3(1), dim3(THREADS), words * 4, p, (uint32_t *)arg_ptr(moved), words));
    BRASA_TRY(brasa_post_launch(cmd, "pages_compact"));
    return copy_pages(cmd, g, p);
}

}  // extern "C"
