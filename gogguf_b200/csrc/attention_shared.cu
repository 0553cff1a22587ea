// Decode attention of a step some of whose rows share a prefix: the prefix's keys and values are read once for all its readers.
//
// With s_j = scale q . k_j, a part over a run of positions is
//     m >= some s_j of the run,   l = sum e^(s_j - m),   O = sum e^(s_j - m) v_j
// and parts add up as O = sum e^(m_i - m) O_i, l alike, whatever the m_i are; the output is O / l.  Two kernels make the parts, side
// by side, so that what computes and what waits for memory share the SMs; a third adds them, always in the same order.
//
// Prefixes: a tile is up to 128 rows of a tensor-core product, members of a group times the query heads of a kv head.  Per page
// of 64 keys S = Q K^T (tcgen05.mma 128 x 64 x 16) lands in tensor memory, four warps take a row per thread, leave P as bfloat16
// where S was and O += P V accumulates in tensor memory, as in the prefill kernel (attention_fast.cu), without its masks: every
// reader sees every key of the prefix.  All (group, tile, kv head)s' pages are one line of work cut into equal runs, one per CTA,
// so that neither the number of readers nor that of kv heads leaves an SM without work, and the grid is the same for every plan:
// a captured step replays with other groups.
//
// A row's own positions: a CTA a (token row, kv head, share), on mma.sync, with the query heads as columns where there are eight
// at most, else as rows, as in the decode kernel of a step without prefixes (attention_fast.cu).  (As rows of the prefix's product, a
// page of a member's own took the tensor core as long as one of the prefix: 64 rows with up to 500 positions of their own on 2,048 were
// 44 us.  As CTAs of the prefix's kernel they ran one an SM: a CTA of a kernel that allocates tensor memory keeps others of it off its
// SM until it has done so.)
//
// Rounding.  P is bfloat16 in front of V, below a maximum that may be an old one, and is summed as it is rounded.  Relative error of
// the output against 64 bits, together / by the kernel for rows alone / of the output's own rounding (10^-3; 64 rows of 32 heads of 128 on 32
// pages, scores of standard deviation 0.5, 1.5, 3, 6): 2.34 2.19 1.91 1.76 / 2.33 1.97 1.70 1.67 / 1.66 all; 16 rows on 512 pages 2.32 2.31 2.11
// 1.82 / 2.30 2.09 1.71 1.66.  The kernel for rows alone has a weight of exactly 1 at the maximum so far, this one does not: summed
// before rounding, that alone was up to 2.4 in steep rows (in a model of both in 64 bits; summed so, 1.8 to 1.9).  The sums as rounded cost nothing
// (64 rows on 512 pages 62.1 us, now 61.7).
//
// What bounds it.  64 rows of 32 heads (8 kv heads of 128) on 512 pages, with up to 200 positions of their own: 62 us (each row by
// itself 700), of which the prefix kernel takes 45 (a page and tile 1.4 us of a CTA, two CTAs an SM; its products alone would take half), the
// rows' own pages behind it 6 more, the parts 5.  Its two tiles ask for 268 MB of pages, of which 134 MB are different: 228 MB come from DRAM,
// 467 MB are read in L2 (ncu, which counts what crosses from one half of L2 to the other twice), so neither is at its rate, and tiles
// side by side, which brought DRAM to 136 MB, took as long.  On 32 pages, with up to 500 positions of their
// own, 28 us (61): the own pages' 74 MB in 17 us (a CTA's beginning and end are worth three of its pages, of which it has one to eight),
// the prefix kernel beside them for the first 10, the parts 3.
// Tried and slower (us, of 64 rows on 32 and 512 pages, when this was 33 and 67): runs in clusters of eight that add up their parts in
// shared memory 40 and 62 (but 17 of 8 rows where this is 12), rows' own pages as rows of the product 74 and 168 or in the line of pages 44
// and 73, own pages as CTAs of the prefix kernel 36 and 64 (24 and 30 of ragged prompts where this was 19 and 20), 128 keys a step 34
// and 70, 256 rows a tile 44 and 73, eight warps for the softmax 37 and 69.  Now: K in three stages 28.7 and 63.4.
#include <climits>
#include <cstring>
#include <initializer_list>
#include <type_traits>

#include "attention_common.cuh"

namespace {

constexpr int ROWS = 128;             // of a tile
constexpr int THREADS = 192;          // of the prefix kernel
constexpr int OWN_THREADS = 128;      // of the kernel over rows' own pages
constexpr int MAX_RUNS = 296;         // of the prefix kernel: two per SM

// Stages of the ring of a row's own pages: 64 KB of them in the form for eight query heads (three CTAs an SM; 96 KB and two: 29.7 us
// where this is 27.9), 96 KB in that for sixteen, whose registers leave room for two.
__host__ __device__ constexpr int own_stages(int stage_bytes, bool eight) {
    const int n = (eight ? 64 : 96) * 1024 / stage_bytes;
    return n < 4 ? n : 4;
}

// The plan, integers of a step, with room for `cap` token rows: how many groups; from word 4 on, per group the place of its first
// member in `rows` (and one place beyond the last group's), its pages and its first member; `rows`, the members' token rows group
// by group; per token row the pages that are its prefix (0: none), its group (-1: none) and its place among the group's
// members; the token rows in the order in which their own pages are read, most pages first.
// A group's members are cut into tiles of equal size; the units of work are the pages of (group, tile, kv head) in that order, and
// run c takes `per` of them from c per on.  The part that run c leaves of a (tile, kv head) begins at row row0 + 128 c, with row0
// the rows of all (tile, kv head)s before: later parts are later in c or in row0, and 128 is the most a part has, so no two
// overlap.
struct SharedArgs {
    const int* plan;
    int cap, runs, shares;            // token rows that the plan has room for; runs; CTAs that share a row's own pages
    float* part_o;                    // dv a row: the prefixes' parts, each [dv / 8][its rows][8], then [token row][query head][share][dv]
    float2* part_ml;                  // [rows]: maximum in log2 units, sum
    int4* where;                      // [token row][kv head]: first row of its prefix's first part, how many parts there are, the
                                      // place of its rows in them, and a part's rows
    int own_row;                      // the first row behind the prefixes' parts
    int max_pages;                    // of a row of the page table: a plan of more is read as one of so many
};

struct SharedPlan {
    const int *count, *first, *pages, *lead, *rows, *pages_of, *group_of, *member_of, *order;
    int cap, max_pages;
    __device__ __forceinline__ SharedPlan(const SharedArgs& a)
        : count(a.plan), first(a.plan + 4), pages(first + a.cap + 1), lead(pages + a.cap), rows(lead + a.cap), pages_of(rows + a.cap),
          group_of(pages_of + a.cap), member_of(group_of + a.cap), order(member_of + a.cap), cap(a.cap), max_pages(a.max_pages) {}
    static __device__ __forceinline__ int tiles(int members, int G) {
        const int most = ROWS / G;
        return (members + most - 1) / most;
    }
    // members of each tile but the last
    static __device__ __forceinline__ int tile_members(int members, int G) {
        const int n = tiles(members, G);
        return (members + n - 1) / n;
    }
    // units of a run: as many for each
    static __device__ __forceinline__ int per(int total, int runs) { return max(1, (total + runs - 1) / runs); }

    // All units, and the group that unit u is of (u < 0: group `which`), by a whole warp: a lane a group.
    struct Group { int before, pages, first, members, lead; };
    // the first of a group's sequences (rows that only fill up a step have none; the others of the group do not need them)
    __device__ __forceinline__ int sequence(const int* seq_of_token, int lead_row, int at, int members) const {
        int b = seq_of_token[lead_row];
        for (int k = 1; b < 0 && k < members; ++k) b = seq_of_token[rows[at + k]];
        return max(b, 0);
    }
    __device__ __forceinline__ Group find(int u, int which, int nkv, int G, int lane, int& total) const {
        Group found = {};
        int groups = 1;
        total = 0;
        for (int g0 = 0; g0 < groups; g0 += 32) {
            const int g = min(g0 + lane, cap - 1);
            // (asked for before the number of groups is known: beyond the last one stands something that is not used)
            const int pg = min(pages[g], max_pages), f = first[g], m = first[g + 1] - f, head = lead[g];
            if (g0 == 0) groups = *count;
            const int units = g0 + lane < groups ? pg * tiles(m, G) * nkv : 0;
            int upto = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            upto += total;
            const bool it = u < 0 ? g0 + lane == which : u >= upto - units && u < upto;
            const unsigned mine = __ballot_sync(0xffffffffu, it && units > 0);
            if (mine != 0) {
                const int from = __ffs(mine) - 1;
                found.before = __shfl_sync(0xffffffffu, upto - units, from);
                found.pages = __shfl_sync(0xffffffffu, pg, from);
                found.first = __shfl_sync(0xffffffffu, f, from);
                found.members = __shfl_sync(0xffffffffu, m, from);
                found.lead = __shfl_sync(0xffffffffu, head, from);
            }
            total = __shfl_sync(0xffffffffu, upto, 31);
        }
        return found;
    }
    // where the parts of a token row and kv head are (see SharedArgs), by a whole warp
    __device__ __forceinline__ int4 where(int tok, int kvh, int nkv, int G, int runs, int lane) const {
        const int which = group_of[tok], mine = member_of[tok];
        if (which < 0) return make_int4(0, 0, 0, 0);
        int total;
        const Group g = find(-1, which, nkv, G, lane, total);
        const int tm = tile_members(g.members, G), p = per(total, runs), tile = mine / tm;
        const int u0 = g.before + (tile * nkv + kvh) * g.pages, c0 = u0 / p, c1 = (u0 + g.pages - 1) / p;
        const int members = min(tm, g.members - tile * tm);
        return make_int4(nkv * G * (g.first + tile * tm) + kvh * G * members + c0 * ROWS, c1 - c0 + 1, (mine - tile * tm) * G, members * G);
    }
};

// 32 bytes, a whole sector, at a time
__device__ __forceinline__ void store8(float* dst, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// What both kinds of CTA are given.
struct SharedStep {
    const bf16* q;
    const int *positions, *seq_of_token, *page_table;
    int max_pages, nq, nkv, d, dv, n_pages;
    float scale_log2;
    int* status;
};

template <int DK, int DV, bool EXACT>
__global__ void __launch_bounds__(256, 2) shared_prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                   const SharedStep st, const SharedArgs args) {
    // (the dynamic segment is the only shared memory and is asked to start on a 1024-byte boundary: two CTAs share an SM)
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int HK = DK / 64, HV = DV / 64;
    const int d = EXACT ? DK : st.d, dv = EXACT ? DV : st.dv, nkv = st.nkv, nq = st.nq, G = nq / nkv;
    const float scale_log2 = st.scale_log2;
    int* status = st.status;
    constexpr int QBOX = ROWS * 64 * 2;             // [64 columns x 128 rows] of Q: 16 KB
    constexpr int KBOX = 64 * 64 * 2;               // [64 columns x 64 keys] of K or V: 8 KB
    constexpr int Q_BYTES = HK * QBOX, K_STAGE = HK * KBOX, V_STAGE = HV * KBOX;
    constexpr int TMEM_COLS = 256;                  // two score buffers of 64 columns, then O
    uint8_t* Qs = smem;
    uint8_t* Ks = Qs + Q_BYTES;                     // two stages
    uint8_t* Vs = Ks + 2 * K_STAGE;                 // two stages
    uint64_t* bars = (uint64_t*)(Vs + 2 * V_STAGE);
    uint64_t* q_full = bars;                        // the four softmax warps have written a run's Q
    uint64_t* k_full = bars + 1;                    // [2]
    uint64_t* k_empty = bars + 3;                   // [2]
    uint64_t* v_full = bars + 5;                    // [2]
    uint64_t* v_empty = bars + 7;                   // [2]
    uint64_t* s_full = bars + 9;                    // [2]
    uint64_t* p_ready = bars + 11;                  // [2] (two in turn: a warp may be a page ahead of another)
    uint64_t* pv_done = bars + 13;
    uint64_t* o_done = bars + 14;                   // every P V of a run's (tile, kv head) is complete
    uint32_t* tmem_slot = (uint32_t*)(bars + 15);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run = (int)blockIdx.x;
    const SharedPlan plan(args);
    int total;
    plan.find(-1, -1, nkv, G, lane, total);
    const int per = plan.per(total, args.runs), u_begin = min(run * per, total), u_end = min(u_begin + per, total);
    // The next kernel's CTAs are let in when q is there, which they need and this kernel's work they do not.
    if (u_begin >= u_end) {
        pdl_wait();
        return;
    }
    if (threadIdx.x == 0) {
        tma::mbar_init(q_full, 4);
        for (int i = 0; i < 2; ++i) {
            tma::mbar_init(&k_full[i], 1); tma::mbar_init(&k_empty[i], 1);
            tma::mbar_init(&v_full[i], 1); tma::mbar_init(&v_empty[i], 1);
            tma::mbar_init(&s_full[i], 1); tma::mbar_init(&p_ready[i], 4);
        }
        tma::mbar_init(pv_done, 1);
        tma::mbar_init(o_done, 1);
        *abort_flag = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&tmK); tma::prefetch_map(&tmV);
    }
    if (warp == 5) tc5::alloc(tmem_slot, TMEM_COLS);
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    const uint32_t S_t = *tmem_slot, O_t = S_t + 128;
    // (a shared-memory base off the 1024-byte boundary would corrupt the swizzled tiles: refuse and say so)
    bool ok = (tma::smem_u32(smem) & 1023u) == 0;
    if (!ok && threadIdx.x == 0) atomicCAS(status, 0, 70);

    // The run is cut where the (tile, kv head) changes.  Every role walks the same cuts.
    struct Piece { int first, members, head, page0, pages, lead, all_first, all_members; size_t row0; };
    auto piece_at = [&](int u) -> Piece {
        int all;
        const SharedPlan::Group g = plan.find(u, -1, nkv, G, lane, all);
        const int tm = plan.tile_members(g.members, G), rel = u - g.before;
        const int th = rel / g.pages, tile = th / nkv;
        Piece r;
        r.head = th - tile * nkv;
        r.page0 = rel - th * g.pages;
        r.pages = min(g.pages - r.page0, u_end - u);
        r.first = g.first + tile * tm;
        r.members = min(tm, g.members - tile * tm);
        r.lead = g.lead;
        r.all_first = g.first;
        r.all_members = g.members;
        r.row0 = (size_t)nkv * G * r.first + (size_t)r.head * G * r.members + (size_t)run * ROWS;
        return r;
    };
    // (a warp goes on or leaves as a whole: what follows a wait is for whole warps)
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) -> bool {
        return __all_sync(0xffffffffu, tma::mbar_wait(bar, phase, abort_flag, status, code));
    };

    if (warp == 5 || (warp == 4 && lane != 0)) { pdl_wait(); pdl_launch(); }
    int j = 0;                                      // pages so far
    if (warp == 4) {
        // The prefix's pages were written by earlier steps (this step's tokens go to pages of the rows' own), so they are
        // streamed before the kernel before this one has finished.
        for (int u = u_begin; u < u_end;) {
            const Piece r = piece_at(u);
            u += r.pages;
            if (lane == 0 && ok) {
                const int* pt = st.page_table + (size_t)plan.sequence(st.seq_of_token, r.lead, r.all_first, r.all_members) * st.max_pages;
                for (int i = 0; i < r.pages; ++i, ++j) {
                    const int s = j & 1;
                    const uint32_t ph = (uint32_t)((j >> 1) & 1) ^ 1u;
                    const int row = (gg_page(pt, r.page0 + i, st.max_pages, PageBounds{st.n_pages, status}, 54) * nkv + r.head) * PAGE;
                    if (!(ok = tma::mbar_wait(&k_empty[s], ph, abort_flag, status, 71))) break;
                    tma::mbar_expect_tx(&k_full[s], K_STAGE);
#pragma unroll
                    for (int hf = 0; hf < HK; ++hf) tma::load_2d(Ks + s * K_STAGE + hf * KBOX, &tmK, &k_full[s], hf * 64, row);
                    if (!(ok = tma::mbar_wait(&v_empty[s], ph, abort_flag, status, 72))) break;
                    tma::mbar_expect_tx(&v_full[s], V_STAGE);
#pragma unroll
                    for (int hf = 0; hf < HV; ++hf) tma::load_2d(Vs + s * V_STAGE + hf * KBOX, &tmV, &v_full[s], hf * 64, row);
                    if (j == 1 || u >= u_end && i + 1 == r.pages) { pdl_wait(); pdl_launch(); }
                }
            }
            __syncwarp();
        }
    } else if (warp == 5) {
        const uint32_t idesc_qk = tc5::idesc_bf16(ROWS, 64, 0), idesc_pv = tc5::idesc_bf16(ROWS, EXACT ? DV : (dv + 15) & ~15, 1);
        // A matrix descriptor's upper word is the same for all; of the lower one an operand's place is added, in 16 bytes.
        const uint64_t dq = tc5::smem_desc(tma::smem_u32(Qs), 16, 1024), dk = tc5::smem_desc(tma::smem_u32(Ks), 16, 1024);
        const uint64_t dw = tc5::smem_desc(tma::smem_u32(Vs), KBOX, 1024);
        auto moved = [](uint64_t desc, uint32_t bytes) -> uint64_t { return desc & 0xffffffff00000000ull | (uint32_t)desc + (bytes >> 4); };
        auto issue_scores = [&](int j) -> bool {
            const int s = j & 1;
            if (!tma::mbar_wait(&k_full[s], (uint32_t)((j >> 1) & 1), abort_flag, status, 73)) return false;
            tc5::fence_after();
            const uint64_t dks = moved(dk, (uint32_t)(s * K_STAGE));
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
                if (!EXACT && ks * 16 >= d) break;
                tc5::mma(S_t + (uint32_t)(s * 64), moved(dq, (uint32_t)((ks >> 2) * QBOX + (ks & 3) * 32)),
                         moved(dks, (uint32_t)((ks >> 2) * KBOX + (ks & 3) * 32)), idesc_qk, ks > 0 ? 1u : 0u);
            }
            tc5::commit(&s_full[s]);
            tc5::commit(&k_empty[s]);
            return true;
        };
        int pieces = 0;
        for (int u = u_begin; u < u_end; ++pieces) {
            const Piece r = piece_at(u);
            u += r.pages;
            if (lane == 0 && ok) {
                // (a piece's first scores come after the last P V of the piece before: its Q is written when that is read)
                ok = tma::mbar_wait(q_full, (uint32_t)(pieces & 1), abort_flag, status, 74);
                if (ok) ok = issue_scores(j);
                for (int i = 0; i < r.pages && ok; ++i, ++j) {
                    // The next page's scores do not wait for this page's softmax: their buffer was last read by the
                    // softmax of page j - 1, whose p_ready this thread has already seen.
                    if (i + 1 < r.pages && !(ok = issue_scores(j + 1))) break;
                    const int s = j & 1;
                    const uint32_t ph = (uint32_t)((j >> 1) & 1);
                    if (!(ok = tma::mbar_wait(&v_full[s], ph, abort_flag, status, 76))) break;
                    if (!(ok = tma::mbar_wait(&p_ready[s], ph, abort_flag, status, 75))) break;
                    tc5::fence_after();
                    const uint64_t dvs = moved(dw, (uint32_t)(s * V_STAGE));
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        // P of page j lies in the first 32 columns of score buffer j & 1: 16 keys are 8 columns
                        tc5::mma_a_tmem(O_t, S_t + (uint32_t)(s * 64 + kk * 8), moved(dvs, (uint32_t)(kk * 2048)), idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
                    tc5::commit(pv_done);
                    tc5::commit(&v_empty[s]);
                }
                if (ok) tc5::commit(o_done);
            }
            __syncwarp();
        }
    } else {
        const int row = threadIdx.x;                           // row of the tile = tensor-memory lane
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        int pieces = 0;
        for (int u = u_begin; u < u_end && ok; ++pieces) {
            const Piece r = piece_at(u);
            u += r.pages;
            const int rows = r.members * G;
            const bool live = row < rows, idle = warp * 32 >= rows;     // (a warp without rows only keeps the pace)
            const int member = live ? row / G : 0;
            const bf16* src = st.q + ((size_t)plan.rows[r.first + member] * nq + (size_t)r.head * G + (row - member * G)) * d;
            if (pieces == 0) { pdl_wait(); pdl_launch(); }     // q, and the scratch is free
            if (!idle) {
                // Q into its swizzled tile: row r of a box is 128 bytes, 16-byte chunk c at place c ^ (r & 7)
#pragma unroll
                for (int c = 0; c < DK / 8; ++c) {
                    const uint4 x = live && (EXACT || c * 8 < d) ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(Qs + (c >> 3) * QBOX + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = x;
                }
            }
            tc5::fence_proxy_async_smem();
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(q_full);
            float m_used = -INFINITY, l = 0.f;
            for (int i = 0; i < r.pages; ++i, ++j) {
                const int s = j & 1;
                if (!(ok = wait(&s_full[s], (uint32_t)((j >> 1) & 1), 77))) break;
                tc5::fence_after();
                if (!idle) {
                    uint32_t sr[64], pk[32];
                    tc5::ld32(S_t + lane_off + (uint32_t)(s * 64), sr);
                    tc5::ld32(S_t + lane_off + (uint32_t)(s * 64) + 32, sr + 32);
                    tc5::wait_ld();
                    // P = 2^(score scale - maximum in use) as bfloat16 pairs; returns the sum of the page's P, as they are rounded: the
                    // maximum in use is an old one, so a row's largest weight is not a power of two, and a row that looks at
                    // one key gets that key's value only where both sums hold the same weight.
                    auto exponentials = [&]() -> float {
                        const float mu = m_used == -INFINITY ? 0.f : m_used;
                        const unsigned long long sc2 = pack2(scale_log2, scale_log2), nmu2 = pack2(-mu, -mu);
                        unsigned long long l4[4] = {pack2(0.f, 0.f), pack2(0.f, 0.f), pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float x0, x1;
                            unpack2(fma2(pack2(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1])), sc2, nmu2), x0, x1);
                            pk[e] = pack_bf16(fast_exp2(x0), fast_exp2(x1));
                            l4[e & 3] = add2(l4[e & 3], pack2(__uint_as_float(pk[e] << 16), __uint_as_float(pk[e] & 0xffff0000u)));
                        }
                        float la, lb;
                        unpack2(add2(add2(l4[0], l4[1]), add2(l4[2], l4[3])), la, lb);
                        return la + lb;
                    };
                    // The maximum in use is that of the pages before (any is exact while nothing overflows): only where a row
                    // has none yet, or the page's sum says that a score lies more than 2^64 above it, is the page's own found, O rescaled where it has grown by more than 2^8, and the page computed again.
                    float lpage = 0.f;
                    bool again = m_used == -INFINITY;
                    if (!__any_sync(0xffffffffu, again)) {
                        lpage = exponentials();
                        again = !(lpage < 1.8446744e19f);
                    }
                    if (__any_sync(0xffffffffu, again)) {
                        float m8[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) m8[k] = __uint_as_float(sr[k]);
#pragma unroll
                        for (int c = 8; c < 64; ++c) m8[c & 7] = fmaxf(m8[c & 7], __uint_as_float(sr[c]));
                        const float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                                               fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7]))) * scale_log2;
                        const bool grow = mx > m_used + 8.0f || (m_used == -INFINITY && mx != -INFINITY);
                        if (__any_sync(0xffffffffu, grow)) {
                            // (a row without a maximum has nothing in O: all its P were 0)
                            const bool had = grow && m_used != -INFINITY;
                            float corr = 1.0f;
                            if (grow) {
                                if (had) corr = fast_exp2(m_used - mx);
                                m_used = mx;
                                l *= corr;
                            }
                            if (i > 0 && __any_sync(0xffffffffu, had)) {
                                // P V of the page before must be complete before O is rescaled (that of this page waits for
                                // this warp's p_ready, that of two pages ago came before these scores: the phase is the one meant)
                                if (!(ok = wait(pv_done, (uint32_t)((j - 1) & 1), 78))) break;
                                tc5::fence_after();
#pragma unroll 1
                                for (int c0 = 0; c0 < (EXACT ? DV : dv); c0 += 32) {
                                    uint32_t o[32];
                                    tc5::ld32(O_t + lane_off + c0, o);
                                    tc5::wait_ld();
#pragma unroll
                                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
                                    tc5::st32(O_t + lane_off + c0, o);
                                }
                                tc5::wait_st();
                            }
                        }
                        lpage = exponentials();
                    }
                    l += lpage;
                    // P over this thread's own row of the scores it has read: nothing else uses this buffer now (the P V of
                    // two pages ago was issued before these scores, and the tensor core works in order)
                    tc5::st32(S_t + lane_off + (uint32_t)(s * 64), pk);
                    tc5::wait_st();
                }
                tc5::fence_before();
                __syncwarp();
                if (lane == 0) tma::mbar_arrive(&p_ready[s]);
            }
            // The last P V (on a barrier of its own: by pv_done's parity, two phases not yet complete would look like the last one
            // being so), then the part
            if (!ok || !(ok = wait(o_done, (uint32_t)(pieces & 1), 79))) break;
            tc5::fence_after();
            if (!idle) {
                // (a lane's 32 bytes lie beside its neighbours', a row's do not: rows in one piece took three times as long to write)
                float* dst = args.part_o + r.row0 * dv + row * 8;
#pragma unroll 1
                for (int c0 = 0; c0 < (EXACT ? DV : dv); c0 += 32) {
                    uint32_t o[32];
                    tc5::ld32(O_t + lane_off + c0, o);
                    tc5::wait_ld();
                    if (live) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            if (EXACT || c0 + c < dv) store8(dst + (size_t)(c0 + c) * rows, o + c);
                    }
                }
                if (live) args.part_ml[r.row0 + row] = make_float2(m_used, l);
                tc5::fence_before();
            }
        }
    }
    pdl_wait();                                     // (every kernel of a step waits for the one before it: common.cuh)
    tc5::fence_before();
    __syncthreads();
    if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }       // let copies in flight land before the CTA goes away
        __syncthreads();
    }
    if (warp == 5) {
        tc5::fence_after();
        tc5::dealloc(S_t, TMEM_COLS);
    }
}

// What a warp holds of a row's own pages: the query heads, the sums so far, and what it does with its 16 keys of a page.  The maximum m is
// in log2 units, l a lane's share of the sum until `finish`.
//
// Up to sixteen query heads are the rows of the products (fragments as in attention_fast.cu).
template <int DK, int DV, bool EXACT>
struct SixteenHeads {
    static constexpr int KS = DK / 16, NT = DV / 8, BOX_BYTES = 64 * 64 * 2;
    uint32_t qa[KS][4];
    float o[NT][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
    __device__ __forceinline__ void load(const bf16* q0, int G, int d, int g, int t) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = g + 8 * (e & 1), c = ks * 16 + 2 * t + 8 * (e >> 1);
                qa[ks][e] = row < G && (EXACT || c < d) ? __ldcg(reinterpret_cast<const unsigned int*>(q0 + (size_t)row * d + c)) : 0u;
            }
    }
    __device__ __forceinline__ void page(const uint8_t* k, const uint8_t* v, int krow, int key0, int pos, float scale_log2, int lane) {
        const int t = lane & 3;
        float sc[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16* box = reinterpret_cast<const bf16*>(k + (ks >> 2) * BOX_BYTES);
            uint32_t kb[4];
            ldsm_x4(kb, sw<64>(const_cast<bf16*>(box), krow + (lane & 7) + ((lane >> 4) << 3), (ks & 3) * 2 + ((lane >> 3) & 1)));
            mma16816(sc[0], qa[ks], kb[0], kb[1]);
            mma16816(sc[1], qa[ks], kb[2], kb[3]);
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = key0 + j * 8 + 2 * t + (e & 1) <= pos ? sc[j][e] * scale_log2 : -INFINITY;
                sc[j][e] = x;
                mx[e >> 1] = fmaxf(mx[e >> 1], x);
            }
        uint32_t pa[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            const float mn = fmaxf(m[r], mx[r]);
            const float mu = mn == -INFINITY ? 0.f : mn;
            const float corr = fast_exp2(m[r] - mu);
            m[r] = mn;
            const float p00 = fast_exp2(sc[0][2 * r] - mu), p01 = fast_exp2(sc[0][2 * r + 1] - mu);
            const float p10 = fast_exp2(sc[1][2 * r] - mu), p11 = fast_exp2(sc[1][2 * r + 1] - mu);
            l[r] = l[r] * corr + (p00 + p01 + p10 + p11);
            pa[r] = pack_bf16(p00, p01);
            pa[2 + r] = pack_bf16(p10, p11);
#pragma unroll
            for (int n = 0; n < NT; ++n) { o[n][2 * r] *= corr; o[n][2 * r + 1] *= corr; }
        }
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
            const bf16* box = reinterpret_cast<const bf16*>(v + (np >> 2) * BOX_BYTES);
            uint32_t vb[4];
            ldsm_x4_trans(vb, sw<64>(const_cast<bf16*>(box), krow + (lane & 7) + (((lane >> 3) & 1) << 3), (np & 3) * 2 + (lane >> 4)));
            mma16816(o[2 * np], pa, vb[0], vb[1]);
            mma16816(o[2 * np + 1], pa, vb[2], vb[3]);
        }
    }
    // a head's values into `row_of(head)`, its maximum and sum into `ml_of(head)`
    template <typename Row, typename Ml>
    __device__ __forceinline__ void finish(int G, int g, int t, Row row_of, Ml ml_of) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        // only the G rows that are query heads go on (the MMA tile has 16)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (g + 8 * r >= G) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(row_of(g + 8 * r) + n * 8 + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
            if (t == 0) *ml_of(g + 8 * r) = make_float2(m[r], l[r]);
        }
    }
};

// Up to eight are the columns instead, S^T = K Q^T and O^T = V^T P^T: half the products and half the registers for O, for P^T's way from
// the rows of one product to those of the other (a transposition of 8 x 8 in registers).
template <int DK, int DV, bool EXACT>
struct EightHeads {
    static constexpr int KS = DK / 16, NT = DV / 16, BOX_BYTES = 64 * 64 * 2;
    uint32_t qb[KS][2];
    float o[NT][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};      // of heads 2 t and 2 t + 1
    __device__ __forceinline__ void load(const bf16* q0, int G, int d, int g, int t) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = ks * 16 + 2 * t + 8 * e;
                qb[ks][e] = g < G && (EXACT || c < d) ? __ldcg(reinterpret_cast<const unsigned int*>(q0 + (size_t)g * d + c)) : 0u;
            }
    }
    static __device__ __forceinline__ uint32_t transposed(uint32_t x) {
        uint32_t y;
        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
        return y;
    }
    __device__ __forceinline__ void page(const uint8_t* k, const uint8_t* v, int krow, int key0, int pos, float scale_log2, int lane) {
        const int g = lane >> 2;
        float sc[4] = {};                                  // keys g, g, g + 8, g + 8; heads 2 t, 2 t + 1, 2 t, 2 t + 1
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16* box = reinterpret_cast<const bf16*>(k + (ks >> 2) * BOX_BYTES);
            uint32_t ka[4];
            ldsm_x4(ka, sw<64>(const_cast<bf16*>(box), krow + (lane & 7) + (((lane >> 3) & 1) << 3), (ks & 3) * 2 + (lane >> 4)));
            mma16816(sc, ka, qb[ks][0], qb[ks][1]);
        }
        float p[4], corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float x0 = key0 + g <= pos ? sc[h] * scale_log2 : -INFINITY, x1 = key0 + g + 8 <= pos ? sc[2 + h] * scale_log2 : -INFINITY;
            float mx = fmaxf(x0, x1);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[h], mx), mu = mn == -INFINITY ? 0.f : mn;
            corr[h] = fast_exp2(m[h] - mu);
            m[h] = mn;
            p[h] = fast_exp2(x0 - mu);
            p[2 + h] = fast_exp2(x1 - mu);
            l[h] = l[h] * corr[h] + (p[h] + p[2 + h]);
        }
        const uint32_t p0 = transposed(pack_bf16(p[0], p[1])), p1 = transposed(pack_bf16(p[2], p[3]));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bf16* box = reinterpret_cast<const bf16*>(v + (n >> 2) * BOX_BYTES);
            uint32_t va[4];
            ldsm_x4_trans(va, sw<64>(const_cast<bf16*>(box), krow + (lane & 7) + ((lane >> 4) << 3), (n & 3) * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= corr[e & 1];
            mma16816(o[n], va, p0, p1);
        }
    }
    template <typename Row, typename Ml>
    __device__ __forceinline__ void finish(int G, int g, int t, Row row_of, Ml ml_of) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (2 * t + h >= G) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                row_of(2 * t + h)[n * 16 + g] = o[n][h];
                row_of(2 * t + h)[n * 16 + g + 8] = o[n][2 + h];
            }
            if (g == 0) *ml_of(2 * t + h) = make_float2(m[h], l[h]);
        }
    }
};

// One share of the pages that only row `tok` reads, for the query heads of one kv head: four warps take 16 keys of every page, their
// results are merged in shared memory; the first thread asks for the pages.  (A warp more for that leaves an SM two CTAs instead of three:
// 64 rows on 32 pages 31 us, this 29.4.)  Rows with many pages come first, so that the last CTAs to begin are short: 27.9 us.
// This kernel starts when the prefix kernel's CTAs have all seen the kernel before them complete, and its last CTA alone waits for the
// prefix kernel, at its end: what it reads, q and the newest position among it, was there when it started.
template <int DK, int DV, bool EXACT, bool EIGHT>
__global__ void __maxnreg__(EIGHT ? 128 : 144) shared_own_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                 const SharedStep st, const SharedArgs args) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const SharedPlan plan(args);
    const int pair = (int)blockIdx.x / args.shares, kvh = pair % st.nkv, share = (int)blockIdx.x % args.shares, tok = plan.order[pair / st.nkv];
    constexpr int HK = DK / 64, HV = DV / 64;
    constexpr int BOX_BYTES = 64 * 64 * 2;                 // 8 KB
    constexpr int STAGE_BYTES = (HK + HV) * BOX_BYTES;     // K halves then V halves
    constexpr int STAGES = own_stages(STAGE_BYTES, EIGHT);
    constexpr int LD = DV + 4;                             // of a merged row: lanes of a warp write to banks of their own
    const int d = EXACT ? DK : st.d, dv = EXACT ? DV : st.dv, nkv = st.nkv, nq = st.nq, G = nq / nkv;
    int* status = st.status;
    uint64_t* full = (uint64_t*)(smem + STAGES * STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    volatile int* abort_flag = (volatile int*)(empty + STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int b = st.seq_of_token[tok], at = st.positions[tok], first = plan.pages_of[tok];
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { tma::mbar_init(&full[s], 1); tma::mbar_init(&empty[s], 4); }
        *abort_flag = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&tmK);
        tma::prefetch_map(&tmV);
    }
    __syncthreads();
    const int pos = b >= 0 ? at : -1;
    int p_begin = 0, npg = 0;
    if (b >= 0) {
        const int n = max(0, pos / PAGE + 1 - first), each = (n + args.shares - 1) / args.shares;
        p_begin = first + share * each;
        npg = max(0, min(each, n - share * each));
    }
    using Heads = std::conditional_t<EIGHT, EightHeads<DK, DV, EXACT>, SixteenHeads<DK, DV, EXACT>>;
    Heads heads;
    int4 where = make_int4(0, 0, 0, 0);
    if (npg > 0) {
        const int* pt = st.page_table + (size_t)b * st.max_pages;
        auto ask = [&](int i) {             // for page i, by one thread
            const int s = i % STAGES;
            tma::mbar_expect_tx(&full[s], STAGE_BYTES);
            const int row = (gg_page(pt, p_begin + i, st.max_pages, PageBounds{st.n_pages, status}, 54) * nkv + kvh) * PAGE;
            uint8_t* dst = smem + s * STAGE_BYTES;
#pragma unroll
            for (int hf = 0; hf < HK; ++hf) tma::load_2d(dst + hf * BOX_BYTES, &tmK, &full[s], hf * 64, row);
#pragma unroll
            for (int hf = 0; hf < HV; ++hf) tma::load_2d(dst + (HK + hf) * BOX_BYTES, &tmV, &full[s], hf * 64, row);
        };
        if (threadIdx.x == 0)
            for (int i = 0; i < min(npg, STAGES); ++i) ask(i);
        __syncwarp();
        heads.load(st.q + ((size_t)tok * nq + (size_t)kvh * G) * d, G, d, g, t);
        if (warp == 3 && share == 0) where = plan.where(tok, kvh, nkv, G, args.runs, lane);
        const int krow = warp * 16;     // this warp's 16 keys of every page
        for (int i = 0; i < npg; ++i) {
            const int s = i % STAGES;
            const uint32_t ph = (uint32_t)(i / STAGES) & 1u;
            if (!__all_sync(0xffffffffu, tma::mbar_wait(&full[s], ph, abort_flag, status, 12))) break;
            const uint8_t* stage = smem + s * STAGE_BYTES;
            const int key0 = (p_begin + i) * PAGE + krow;
            // (a decision of the whole warp: any visible key among these 16?)
            if (key0 <= pos) heads.page(stage, stage + HK * BOX_BYTES, krow, key0, pos, st.scale_log2, lane);
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&empty[s]);
            if (threadIdx.x == 0 && i + STAGES < npg && tma::mbar_wait(&empty[s], ph, abort_flag, status, 11)) ask(i + STAGES);
            __syncwarp();
        }
    } else if (warp == 3 && share == 0) {
        where = plan.where(tok, kvh, nkv, G, args.runs, lane);
    }
    __syncthreads();          // all pages consumed (or the CTA gave up): the ring can be reused for the merge
    if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }       // let copies in flight land before the CTA goes away
        __syncthreads();
    }
    if (warp == 3 && share == 0 && lane == 0) args.where[tok * nkv + kvh] = where;
    float* sm_o = reinterpret_cast<float*>(smem);                 // [4][16][LD]
    float2* sm_ml = reinterpret_cast<float2*>(sm_o + 4 * 16 * LD);     // [4][16]
    heads.finish(G, g, t, [&](int head) { return sm_o + (warp * 16 + head) * LD; }, [&](int head) { return sm_ml + warp * 16 + head; });
    __syncthreads();
    for (int idx = threadIdx.x; idx < G * dv / 4; idx += OWN_THREADS) {
        const int r = idx / (dv / 4), c = (idx - r * (dv / 4)) * 4;
        float2 ml[4];
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) { ml[w] = sm_ml[w * 16 + r]; M = fmaxf(M, ml[w].x); }
        if (M != -INFINITY) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = fast_exp2(ml[w].x - M);
                const float4 v = *reinterpret_cast<const float4*>(&sm_o[(w * 16 + r) * LD + c]);
                L = fmaf(ml[w].y, f, L);
                acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
            }
        }
        const size_t to = (size_t)args.own_row + ((size_t)tok * nq + (size_t)kvh * G + r) * args.shares + share;
        *reinterpret_cast<float4*>(args.part_o + to * dv + c) = acc;
        if (c == 0) args.part_ml[to] = make_float2(M, L);
    }
    pdl_launch();
    // The end of this kernel is the prefix kernel's end, too, for the kernel after it: one CTA that waits for it is enough, and the
    // others leave their place to those that have not begun.
    if (blockIdx.x == gridDim.x - 1) pdl_wait();
}

// Half a warp a row, eight columns a lane, or several (`team`, a power of two): its prefix's parts in the order of their runs, then its
// own, each half warp every team-th, then the half warps' sums in their order.
constexpr int JOIN_HALVES = 16;
__global__ void __launch_bounds__(JOIN_HALVES * 16) shared_join_kernel(bf16* __restrict__ out, const int* __restrict__ seq_of_token, int ntok, int nq,
                                                                       int nkv, int team, const float* __restrict__ sink, float out_scale,
                                                                       const AttnShape sh, const SharedArgs args) {
    __shared__ __align__(16) float sm_o[JOIN_HALVES][16][8];
    __shared__ float2 sm_ml[JOIN_HALVES];
    pdl_launch();
    const int lane = threadIdx.x & 15, half = threadIdx.x >> 4, w = half & (team - 1), dv = sh.dv, c = 8 * lane;
    const int row = ((int)blockIdx.x * JOIN_HALVES + half) / team, G = nq / nkv;
    const bool in = row < ntok * nq;
    const int tok = in ? row / nq : 0, h = row - tok * nq;
    const bool real = in && seq_of_token[tok] >= 0;
    pdl_wait();
    float M = -INFINITY, L = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    auto add = [&](float2 ml, const float4& a, const float4& b) {
        const float top = fmaxf(M, ml.x);
        if (top == -INFINITY) return;
        const float f = fast_exp2(M - top), g = fast_exp2(ml.x - top);
        M = top;
        L = fmaf(ml.y, g, L * f);
        acc[0] = fmaf(a.x, g, acc[0] * f); acc[1] = fmaf(a.y, g, acc[1] * f); acc[2] = fmaf(a.z, g, acc[2] * f); acc[3] = fmaf(a.w, g, acc[3] * f);
        acc[4] = fmaf(b.x, g, acc[4] * f); acc[5] = fmaf(b.y, g, acc[5] * f); acc[6] = fmaf(b.z, g, acc[6] * f); acc[7] = fmaf(b.w, g, acc[7] * f);
    };
    if (real) {
        const int4 at = args.where[tok * nkv + h / G];
        const int n = at.y + args.shares, r = at.z + h % G;
        for (int k0 = w; k0 < n; k0 += 4 * team) {
            float2 ml[4];
            float4 a[4], b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = k0 + k * team;
                ml[k] = make_float2(-INFINITY, 0.f);
                a[k] = b[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < n) {
                    const size_t own = (size_t)args.own_row + (size_t)row * args.shares + (i - at.y), part = (size_t)at.x + (size_t)i * ROWS;
                    ml[k] = args.part_ml[i < at.y ? part + r : own];
                    const float4* src = reinterpret_cast<const float4*>(args.part_o + (i < at.y ? part * dv + ((size_t)lane * at.w + r) * 8 : own * dv + c));
                    if (c < dv) { a[k] = src[0]; b[k] = src[1]; }
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) add(ml[k], a[k], b[k]);
        }
    }
    if (team > 1) {
        float4* mine = reinterpret_cast<float4*>(sm_o[half][lane]);
        mine[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        mine[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        if (lane == 0) sm_ml[half] = make_float2(M, L);
        __syncthreads();
        for (int k = 1; w == 0 && k < team; ++k) {
            const float4* theirs = reinterpret_cast<const float4*>(sm_o[half + k][lane]);
            add(sm_ml[half + k], theirs[0], theirs[1]);
        }
    }
    if (w != 0 || !in || c >= dv) return;
    L = attn_sink_sum(L, M, sink, h);
    const float inv = L > 0.f ? out_scale / L : 0.f;
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        y[e] = pack_bf16(attn_gate(acc[2 * e] * inv, sh, tok, h * dv + c + 2 * e), attn_gate(acc[2 * e + 1] * inv, sh, tok, h * dv + c + 2 * e + 1));
    *reinterpret_cast<uint4*>(out + ((size_t)tok * nq + h) * dv + c) = make_uint4(y[0], y[1], y[2], y[3]);
}

template <int DK, int DV, bool EXACT, bool EIGHT>
int launch_shared(const CUtensorMap& tk, const CUtensorMap& tv, int ntok, const SharedStep& st, const SharedArgs& args, cudaStream_t stream) {
    // Q, K x 2, V x 2 (boxes of 64 columns: 16 KB of Q, 8 KB of K or V), barriers
    constexpr int smem = (DK / 64) * (16384 + 2 * 8192) + (DV / 64) * 2 * 8192 + 256;
    // the ring of a row's own pages, over which its warps' results are merged; barriers
    constexpr int stage = (DK + DV) / 64 * 8192, ring = own_stages(stage, EIGHT) * stage, own = ring + 256;
    static_assert(own >= 4 * 16 * (DV + 4 + 2) * 4, "the merge lies where the ring was");
    static int known[2][GG_MAX_DEVICES];
    int resident = 0, rc;
    if ((rc = gg_resident(shared_prefix_kernel<DK, DV, EXACT>, THREADS, smem, known[0], resident)) != 0) return rc;
    if ((rc = gg_resident(shared_own_kernel<DK, DV, EXACT, EIGHT>, OWN_THREADS, own, known[1], resident)) != 0) return rc;
    if ((rc = gg_launch(shared_prefix_kernel<DK, DV, EXACT>, dim3(args.runs), dim3(THREADS), smem, stream, 1, tk, tv, st, args)) != 0) return rc;
    return gg_launch(shared_own_kernel<DK, DV, EXACT, EIGHT>, dim3(ntok * st.nkv * args.shares), dim3(OWN_THREADS), own, stream, 1, tk, tv, st, args);
}

}  // namespace

// Decode attention (see gg_attn_decode_tma) of a step with shared prefixes: plan as at SharedArgs; runs (1 to 296): CTAs over
// the prefixes; shares (1 to 64): CTAs that share a row's own pages; part: scratch of (nq ntok (1 + shares) + 128 runs) (dv + 2) + 4
// ntok nkv floats, on a 32-byte boundary.
// status: codes 71-79 (prefixes), 11 and 12 (own pages) name the wait that ran out; 70: shared memory off its boundary.
//
// The arguments come packed, eight bytes each (see gg_shape_logits).
struct SharedCall {
    const void *q, *k_pool, *v_pool;
    void* out;
    const int *positions, *seq_of_token, *page_table;
    long long max_pages, page_size, n_pages;
    const int* plan;
    long long ntok, nq, nkv, d, dv, runs, shares;
    const float* sink;
    const void* gate;
    long long ldg;
    float* part;
    long long part_floats;
    int* status;
    double scale, out_scale;
};
static_assert(sizeof(SharedCall) == 26 * 8, "as the caller packs it");

GG_API gg_attn_decode_shared(const void* call, cudaStream_t stream) {
    SharedCall c;
    memcpy(&c, call, sizeof(c));
    if (c.ntok <= 0) return 0;
    for (long long n : {c.max_pages, c.n_pages, c.ntok, c.nq, c.nkv, c.ntok * c.nq})
        if (n <= 0 || n > INT_MAX) return GG_ERR_ARG;
    const void *q = c.q, *k_pool = c.k_pool, *v_pool = c.v_pool, *gate = c.gate;
    void* out = c.out;
    const int *positions = c.positions, *seq_of_token = c.seq_of_token, *page_table = c.page_table, *plan = c.plan;
    const int max_pages = (int)c.max_pages, page_size = (int)c.page_size, n_pages = (int)c.n_pages, ntok = (int)c.ntok, nq = (int)c.nq,
              nkv = (int)c.nkv, d = (int)c.d, dv = (int)c.dv, runs = (int)c.runs, shares = (int)c.shares;
    const float *sink = c.sink, scale = (float)c.scale, out_scale = (float)c.out_scale;
    const long long ldg = c.ldg, part_floats = c.part_floats;
    float* part = c.part;
    int* status = c.status;
    if (page_size != PAGE || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > 16 || !attn_shape_ok(d, dv, 0, gate, ldg) || shares < 1 || shares > 64 || runs < 1 || runs > MAX_RUNS ||
        n_pages <= 0 || max_pages <= 0 || status == nullptr || plan == nullptr)
        return GG_ERR_ARG;
    if ((((uintptr_t)q) & 15) || (((uintptr_t)k_pool) & 15) || (((uintptr_t)v_pool) & 15) || (((uintptr_t)out) & 15) || (((uintptr_t)part) & 31))
        return GG_ERR_ARG;
    const long long prefix_rows = (long long)nq * ntok + (long long)ROWS * runs, rows = prefix_rows + (long long)nq * ntok * shares;
    if (part == nullptr || part_floats < rows * (dv + 2) + 4ll * ntok * nkv || rows > 0x7fffffffll) return GG_ERR_ARG;
    // (units, blocks and the rows of the pools are counted in 32 bits: a row lists at most max_pages pages)
    const unsigned long long pool_rows = (unsigned long long)n_pages * nkv * PAGE;
    if (pool_rows > 0x7fffffffull || (unsigned long long)ntok * max_pages * nkv > 0x7fffffffull || (long long)ntok * nkv * shares > 0x3fffffffll)
        return GG_ERR_ARG;
    CUtensorMap tk, tv;
    int rc;
    if ((rc = tma::make_map_bf16(&tk, k_pool, pool_rows, d, d, PAGE)) != 0) return rc;
    if ((rc = tma::make_map_bf16(&tv, v_pool, pool_rows, dv, dv, PAGE)) != 0) return rc;
    const SharedStep st = {(const bf16*)q, positions, seq_of_token, page_table, max_pages, nq, nkv, d, dv, n_pages, scale * 1.4426950408889634f,
                           status};
    float* where = part + rows * dv;
    const SharedArgs args = {plan, ntok, runs, shares, part, reinterpret_cast<float2*>(where + 4ll * ntok * nkv), reinterpret_cast<int4*>(where),
                             (int)prefix_rows, max_pages};
#define GG_SHARED(DK_, DV_, EX_) (nq / nkv <= 8 ? launch_shared<DK_, DV_, EX_, true>(tk, tv, ntok, st, args, stream) \
                                                : launch_shared<DK_, DV_, EX_, false>(tk, tv, ntok, st, args, stream))
    if (d == 128 && dv == 128) rc = GG_SHARED(128, 128, true);
    else if (d == 64 && dv == 64) rc = GG_SHARED(64, 64, true);
    else if (d <= 64 && dv <= 64) rc = GG_SHARED(64, 64, false);
    else if (d <= 64) rc = GG_SHARED(64, 128, false);
    else if (dv <= 64) rc = GG_SHARED(128, 64, false);
    else rc = GG_SHARED(128, 128, false);
#undef GG_SHARED
    if (rc != 0) return rc;
    const AttnShape sh = {d, dv, 0, (const bf16*)gate, ldg};
    // half warps a row: as many as give each SM four CTAs of 16, at most (a part read behind another takes 1 us longer)
    int team = 1;
    while (team < JOIN_HALVES && (long long)ntok * nq * team * 2 <= 148 * 4 * JOIN_HALVES) team *= 2;
    const long long halves = (long long)ntok * nq * team;
    return gg_launch(shared_join_kernel, dim3((unsigned)((halves + JOIN_HALVES - 1) / JOIN_HALVES)), dim3(JOIN_HALVES * 16), 0, stream, 1, (bf16*)out,
                     seq_of_token, ntok, nq, nkv, team, sink, out_scale, sh, args);
}

// 1 if this library was built with checked page tables (the debug build), else 0.
GG_API gg_attention_shared_checked() { return gg_debug_bounds(); }
