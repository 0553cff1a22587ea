// Decode attention of a step some of whose rows share a prefix: every page of the cache that the step's rows read is read once
// per kv head, whoever reads it.
//
// The step's rows are cut into tiles: members of one group (rows that share their first pages), or rows that share nothing, at
// most two halves of 128 rows of a tensor-core product, members times the query heads of a kv head.  What a tile reads is a list
// of units, the pages of its prefix and then, member by member, the pages that are a member's own.  The units of all (tile, kv
// head)s are one line of work cut into equal runs, one per SM, so that neither the number of readers nor that of kv heads
// leaves an SM without work, and the grid is the same for every plan: a captured step replays with other groups.
//
// Per unit of 64 keys and half S = Q K^T (tcgen05.mma 128 x 64 x 16) lands in tensor memory; four warps take a row per thread,
// leave P as bfloat16 where S was (0 where the row does not see the key: all rows see the prefix, a member's rows its own
// pages), and O += P V accumulates in tensor memory.  Both halves use the K and V that were read once.  What a run leaves of a
// row is a part: with s_j = scale q . k_j,
//     m >= some s_j of the run,   l = sum e^(s_j - m),   O = sum e^(s_j - m) v_j
// and parts add up as O = sum e^(m_i - m) O_i, l alike, whatever the m_i are; a second kernel, a warp a row, adds them in the
// order of their runs and writes O / l.
#include "attention_common.cuh"

namespace {

constexpr int CTAS = 148;             // runs: one per SM
constexpr int HALF = 128;             // rows of a half
constexpr int ROWS = 2 * HALF;        // of a tile, at most
constexpr int MAX_TOKENS = 1024;
constexpr int THREADS = 320;          // four warps a half, the producer, the issuer

// The plan, integers of a step, with room for `cap` token rows: how many groups; from word 4 on, per group the place of its first
// member in `rows` (and one place beyond the last group's); its pages that all members share (0: rows that share nothing); `rows`,
// the members' token rows group by group: every token row of the step is in one group; and per member its group's pages.
struct SharedArgs {
    const int* plan;
    int cap;
    float* part_o;                    // [rows][dv]
    int4* where;                      // [token row][kv head]: row of part 0, (first, last) run of the prefix, of its own pages
    float2* part_ml;                  // [rows]: maximum in log2 units, sum
};
// The part that run c leaves of row r of member i of a (tile, kv head) is row row0 + ROWS c + i G + r, with row0 the rows of all
// (tile, kv head)s before: later parts are later in c or in row0, and ROWS is the most a part has, so no two overlap.

// What all roles look up, in the members' order: token rows, sequences, positions, and the own pages of the members before; the
// groups' first members and pages.
struct Table {
    int tok[MAX_TOKENS], seq[MAX_TOKENS], pos[MAX_TOKENS], before[MAX_TOKENS + 1], first[MAX_TOKENS + 1], pages[MAX_TOKENS], warp_sum[THREADS / 32];
};

// A run's share of a (tile, kv head).
struct Run {
    int first, members, a;            // the tile's members, and those of its first half
    int head, prefix;                 // kv head; pages that all members read
    int unit0, units;                 // units of the (tile, kv head) that are this run's
    int start;                        // the (tile, kv head)'s first unit among all
    size_t row0;
};

// 32 bytes, a whole sector, at a time
__device__ __forceinline__ void store8(float* dst, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <int DK, int DV, bool EXACT>
__global__ void __launch_bounds__(THREADS) attn_shared_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const bf16* q, const int* __restrict__ positions,
    const int* __restrict__ seq_of_token, const int* __restrict__ page_table, int max_pages, int nq, int nkv, float scale_log2, int n_pages,
    int* __restrict__ status, int d_, int dv_, const SharedArgs args) {
    constexpr int HK = DK / 64, HV = DV / 64;
    const int d = EXACT ? DK : d_, dv = EXACT ? DV : dv_;
    constexpr int QBOX = HALF * 64 * 2;             // [64 columns x 128 rows] of Q: 16 KB
    constexpr int KBOX = 64 * 64 * 2;               // [64 columns x 64 keys] of K or V: 8 KB
    constexpr int Q_HALF = HK * QBOX, K_STAGE = HK * KBOX, V_STAGE = HV * KBOX;
    constexpr int STAGES = 128 * 1024 / (K_STAGE + V_STAGE);
    constexpr int TMEM_COLS = 512;                  // two score buffers of 64 columns a half, then O of 128 columns a half
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* Qs = smem;
    uint8_t* Ks = Qs + 2 * Q_HALF;
    uint8_t* Vs = Ks + STAGES * K_STAGE;
    uint64_t* bars = (uint64_t*)(Vs + STAGES * V_STAGE);
    uint64_t* q_full = bars;                        // [2] a half's four warps have written a run's Q
    uint64_t* s_full = bars + 2;                    // [2][2] scores of a half, two buffers
    uint64_t* p_ready = bars + 6;                   // [2][2] (two in turn: a warp may be a page ahead of another)
    uint64_t* pv_done = bars + 10;                  // [2]
    uint64_t* o_done = bars + 12;                   // [2] every P V of a run is complete
    uint64_t* k_full = bars + 14;
    uint64_t* k_empty = k_full + STAGES;
    uint64_t* v_full = k_empty + STAGES;
    uint64_t* v_empty = v_full + STAGES;
    uint32_t* tmem_slot = (uint32_t*)(v_empty + STAGES);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    Table* table = reinterpret_cast<Table*>(bars + 64);
    static_assert(14 + 4 * STAGES + 1 <= 64, "the barriers' room");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = nq / nkv, cap = args.cap;
    pdl_launch();                                   // (the whole grid is resident at once: the rule in common.cuh)
    {
        // the table: a thread's members lie side by side
        const int *first = args.plan + 4, *pages = first + cap + 1, *rows = pages + cap, *shared = rows + cap;
        const int each = (cap + THREADS - 1) / THREADS, i0 = (int)threadIdx.x * each;
        int own = 0;
        for (int i = i0; i < min(i0 + each, cap); ++i) {
            const int tok = rows[i], pg = shared[i];
            table->first[i] = first[i];
            table->pages[i] = pages[i];
            const int seq = seq_of_token[tok], pos = positions[tok];
            table->tok[i] = tok; table->seq[i] = seq; table->pos[i] = pos;
            own += seq >= 0 ? max(0, pos / PAGE + 1 - pg) : 0;
            table->before[i + 1] = own;
        }
        if (threadIdx.x == 0) { table->first[cap] = first[cap]; table->before[0] = 0; }
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) table->warp_sum[warp] = upto;
        __syncthreads();
        int add = upto - own;
        for (int w = 0; w < warp; ++w) add += table->warp_sum[w];
        for (int i = i0; i < min(i0 + each, cap); ++i) table->before[i + 1] += add;
    }
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            tma::mbar_init(&q_full[t], 4); tma::mbar_init(&pv_done[t], 1); tma::mbar_init(&o_done[t], 1);
            for (int i = 0; i < 2; ++i) { tma::mbar_init(&s_full[2 * t + i], 1); tma::mbar_init(&p_ready[2 * t + i], 4); }
        }
        for (int i = 0; i < STAGES; ++i) {
            tma::mbar_init(&k_full[i], 1); tma::mbar_init(&k_empty[i], 1);
            tma::mbar_init(&v_full[i], 1); tma::mbar_init(&v_empty[i], 1);
        }
        *abort_flag = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&tmK); tma::prefetch_map(&tmV);
    }
    __syncthreads();
    const int groups = args.plan[0], half = HALF / G;
    auto tiles_of = [&](int g) -> int { return (table->first[g + 1] - table->first[g] + 2 * half - 1) / (2 * half); };
    int total = table->before[cap] * nkv;
    for (int g = 0; g < groups; ++g) total += table->pages[g] * tiles_of(g) * nkv;
    const int per = (total + CTAS - 1) / CTAS, u_begin = min((int)blockIdx.x * per, total), u_end = min(u_begin + per, total);
    if (u_begin >= u_end) {                         // (every kernel of a step waits for the one before it, too)
        pdl_wait();
        return;
    }
    // the part of the run that begins with unit u
    auto run_at = [&](int u) -> Run {
        Run r = {};
        int start = 0;
        for (int g = 0; g < groups; ++g) {
            const int f = table->first[g], m = table->first[g + 1] - f, nt = tiles_of(g), size = (m + nt - 1) / nt, pg = table->pages[g];
            for (int at = 0; at < m; at += size) {
                const int mm = min(size, m - at), n = pg + table->before[f + at + mm] - table->before[f + at];
                if (u < start + n * nkv) {
                    r.first = f + at;
                    r.members = mm;
                    r.a = mm <= half ? mm : (mm + 1) / 2;
                    r.head = (u - start) / n;
                    r.prefix = pg;
                    r.start = start + r.head * n;
                    r.unit0 = u - r.start;
                    r.units = min(n - r.unit0, u_end - u);
                    r.row0 = (size_t)nkv * G * r.first + (size_t)r.head * G * mm;
                    return r;
                }
                start += n * nkv;
            }
        }
        return r;                                   // (not reached: u is below the total)
    };
    // own pages of the tile's members before its member i
    auto before = [&](const Run& r, int i) -> int { return table->before[r.first + i] - table->before[r.first]; };
    // the member whose own page unit u >= prefix is (the last one that begins at or before it)
    auto member_of = [&](const Run& r, int u) -> int {
        int lo = 0, hi = r.members - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (before(r, mid) <= u - r.prefix) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    // whether a run has units of a half's rows
    auto uses = [&](const Run& r, int t) -> bool {
        const int from = t == 0 ? 0 : r.a, to = t == 0 ? r.a : r.members;
        if (from == to) return false;
        if (r.unit0 < r.prefix) return true;
        return max(r.unit0, r.prefix + before(r, from)) < min(r.unit0 + r.units, r.prefix + before(r, to));
    };

    if (warp == 9) tc5::alloc(tmem_slot, TMEM_COLS);
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    const uint32_t tmem = *tmem_slot;
    // (a shared-memory base off the 1024-byte boundary would corrupt the swizzled tiles: refuse and say so)
    bool ok = (tma::smem_u32(smem) & 1023u) == 0;
    if (!ok && threadIdx.x == 0) atomicCAS(status, 0, 29);

    if (warp == 8) {
        // Pages that end before a member's newest position were written by earlier steps, so they are streamed before the kernel
        // before this one has finished.
        if (lane == 0 && ok) {
            int j = 0;
            bool waited = false;
            for (int u = u_begin; u < u_end && ok;) {
                const Run r = run_at(u);
                int member = 0, end = r.prefix;     // the member whose own pages reach up to unit `end`
                for (int i = 0; i < r.units; ++i, ++j) {
                    int page = r.unit0 + i;
                    if (page >= end) { member = member_of(r, page); end = r.prefix + before(r, member + 1); }
                    if (page >= r.prefix) {
                        page -= before(r, member);
                        if (!waited && page >= table->pos[r.first + member] / PAGE) { pdl_wait(); waited = true; }
                    }
                    const int s = j % STAGES;
                    const uint32_t ph = (uint32_t)(j / STAGES & 1) ^ 1u;
                    const int* pt = page_table + (size_t)max(table->seq[r.first + member], 0) * max_pages;
                    const int row = (gg_page(pt, page, max_pages, PageBounds{n_pages, status}, 54) * nkv + r.head) * PAGE;
                    if (!(ok = tma::mbar_wait(&k_empty[s], ph, abort_flag, status, 71))) break;
                    tma::mbar_expect_tx(&k_full[s], K_STAGE);
#pragma unroll
                    for (int hf = 0; hf < HK; ++hf) tma::load_2d(Ks + s * K_STAGE + hf * KBOX, &tmK, &k_full[s], hf * 64, row);
                    if (!(ok = tma::mbar_wait(&v_empty[s], ph, abort_flag, status, 72))) break;
                    tma::mbar_expect_tx(&v_full[s], V_STAGE);
#pragma unroll
                    for (int hf = 0; hf < HV; ++hf) tma::load_2d(Vs + s * V_STAGE + hf * KBOX, &tmV, &v_full[s], hf * 64, row);
                }
                u += r.units;
            }
        }
    } else if (warp == 9) {
        if (lane == 0 && ok) {
            const uint32_t idesc_qk = tc5::idesc_bf16(HALF, 64, 0), idesc_pv = tc5::idesc_bf16(HALF, EXACT ? DV : (dv + 15) & ~15, 1);
            // A matrix descriptor's upper word is the same for all; of the lower one an operand's place is added, in 16 bytes.  (The
            // one thread that issues is what a unit waits for most: 12 products of a half in 1,000 cycles instead of 1,450.)
            const uint64_t dq = tc5::smem_desc(tma::smem_u32(Qs), 16, 1024), dk = tc5::smem_desc(tma::smem_u32(Ks), 16, 1024);
            const uint64_t dw = tc5::smem_desc(tma::smem_u32(Vs), KBOX, 1024);
            auto moved = [](uint64_t desc, uint32_t bytes) -> uint64_t { return desc & 0xffffffff00000000ull | (uint32_t)desc + (bytes >> 4); };
            int j = 0, scored[2] = {0, 0}, done[2] = {0, 0}, runs[2] = {0, 0};
            for (int u = u_begin; u < u_end && ok;) {
                const Run r = run_at(u);
                int reader = 0, end = r.prefix;
                // the halves (bits) that unit i of this run's is for
                auto halves = [&](int i) -> int {
                    const int x = r.unit0 + i;
                    if (x < r.prefix) return r.a < r.members ? 3 : 1;
                    if (x >= end) { reader = member_of(r, x); end = r.prefix + before(r, reader + 1); }
                    return reader < r.a ? 1 : 2;
                };
                auto issue_scores = [&](int j, int bits) -> bool {
                    const int s = j % STAGES;
                    if (!tma::mbar_wait(&k_full[s], (uint32_t)(j / STAGES & 1), abort_flag, status, 73)) return false;
                    tc5::fence_after();
                    const uint64_t dks = moved(dk, (uint32_t)(s * K_STAGE));
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!(bits >> t & 1)) continue;
                        const int b = scored[t] & 1;
                        const uint32_t to = tmem + (uint32_t)(t * 128 + b * 64);
#pragma unroll
                        for (int ks = 0; ks < DK / 16; ++ks) {
                            if (!EXACT && ks * 16 >= d) break;
                            tc5::mma(to, moved(dq, (uint32_t)(t * Q_HALF + (ks >> 2) * QBOX + (ks & 3) * 32)),
                                     moved(dks, (uint32_t)((ks >> 2) * KBOX + (ks & 3) * 32)), idesc_qk, ks > 0 ? 1u : 0u);
                        }
                        tc5::commit(&s_full[2 * t + b]);
                        ++scored[t];
                    }
                    tc5::commit(&k_empty[s]);
                    return true;
                };
                const bool in[2] = {uses(r, 0), uses(r, 1)};
                bool first[2] = {true, true};
                for (int t = 0; t < 2 && ok; ++t)
                    if (in[t]) ok = tma::mbar_wait(&q_full[t], (uint32_t)(runs[t] & 1), abort_flag, status, 74);
                int bits = halves(0);
                if (ok) ok = issue_scores(j, bits);
                for (int i = 0; i < r.units && ok; ++i, ++j) {
                    // The next unit's scores do not wait for this one's softmax: a half's buffer was last read by the softmax of
                    // its page before the last, whose p_ready this thread has already seen.
                    int next = 0;
                    if (i + 1 < r.units) {
                        next = halves(i + 1);
                        if (!(ok = issue_scores(j + 1, next))) break;
                    }
                    const int s = j % STAGES;
                    if (!(ok = tma::mbar_wait(&v_full[s], (uint32_t)(j / STAGES & 1), abort_flag, status, 76))) break;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!(bits >> t & 1) || !ok) continue;
                        const int b = done[t] & 1;
                        if (!(ok = tma::mbar_wait(&p_ready[2 * t + b], (uint32_t)(done[t] >> 1 & 1), abort_flag, status, 75))) continue;
                        tc5::fence_after();
                        const uint64_t dvs = moved(dw, (uint32_t)(s * V_STAGE));
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            // P lies in the first 32 columns of its score buffer: 16 keys are 8 columns
                            tc5::mma_a_tmem(tmem + 256u + (uint32_t)(t * 128), tmem + (uint32_t)(t * 128 + b * 64 + kk * 8),
                                            moved(dvs, (uint32_t)(kk * 2048)), idesc_pv, (!first[t] || kk > 0) ? 1u : 0u);
                        first[t] = false;
                        tc5::commit(&pv_done[t]);
                        ++done[t];
                    }
                    if (!ok) break;
                    tc5::commit(&v_empty[s]);
                    bits = next;
                }
                for (int t = 0; t < 2 && ok; ++t)
                    if (in[t]) { tc5::commit(&o_done[t]); ++runs[t]; }
                u += r.units;
            }
        }
    } else {
        const int t = warp >> 2, row = (int)threadIdx.x & (HALF - 1);       // half; row of it = tensor-memory lane
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16, S_t = tmem + (uint32_t)(t * 128), O_t = tmem + 256u + (uint32_t)(t * 128);
        // (a warp goes on or leaves as a whole: what follows a wait is for whole warps)
        auto wait = [&](uint64_t* bar, uint32_t phase, int code) -> bool {
            return __all_sync(0xffffffffu, tma::mbar_wait(bar, phase, abort_flag, status, code));
        };
        int n = 0, runs = 0;                               // pages of this half so far, and runs
        bool waited = false;
        for (int u = u_begin; u < u_end && ok;) {
            const Run r = run_at(u);
            u += r.units;
            const bool in = uses(r, t);
            if (!waited) { pdl_wait(); waited = true; }        // q, and the scratch is free
            // where the second kernel finds the members' parts
            auto note = [&]() {
                for (int i = row; i < r.members; i += HALF) {
                    const int b = r.start + r.prefix + before(r, i), e = r.start + r.prefix + before(r, i + 1) - 1;
                    const int p0 = r.start / per, p1 = r.prefix > 0 ? (r.start + r.prefix - 1) / per : p0 - 1;
                    const int o0 = e >= b ? max(b / per, p1 + 1) : 0, o1 = e >= b ? e / per : -1;
                    args.where[table->tok[r.first + i] * nkv + r.head] = make_int4((int)r.row0 + i * G, p0, p1 - p0 + 1, o0 | max(0, o1 - o0 + 1) << 16);
                }
            };
            const bool notes = t == 0 && r.unit0 == 0;
            if (!in) {
                if (notes) note();
                continue;
            }
            const int base = t == 0 ? 0 : r.a, rows = (t == 0 ? r.a : r.members - r.a) * G;
            const int member = base + row / G;                 // (rows behind the last member's see nothing)
            const bool idle = (warp & 3) * 32 >= rows;         // (a warp without rows only keeps the pace)
            const int lo = base + (warp & 3) * 32 / G, hi = base + ((warp & 3) * 32 + 31) / G;     // members of this warp's rows
            if (!idle) {
                // Q into its swizzled tile: row r of a box is 128 bytes, 16-byte chunk c at place c ^ (r & 7)
                const bf16* src = q + ((size_t)table->tok[r.first + (row < rows ? member : base)] * nq + (size_t)r.head * G + row % G) * d;
#pragma unroll
                for (int c = 0; c < DK / 8; ++c) {
                    const uint4 x = row < rows && (EXACT || c * 8 < d) ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(Qs + t * Q_HALF + (c >> 3) * QBOX + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = x;
                }
            }
            tc5::fence_proxy_async_smem();
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&q_full[t]);
            if (notes) note();                                 // (while the first scores are made)
            float m_used = -INFINITY, l = 0.f;
            int reader = -1, end = r.prefix;                   // the member whose own pages reach up to unit `end` (-1: all read)
            bool fresh = true;                                 // no P V of this run yet
            for (int i = 0; i < r.units && ok; ++i) {
                const int x = r.unit0 + i;
                if (x >= end) { reader = member_of(r, x); end = r.prefix + before(r, reader + 1); }
                if (reader >= 0 && (reader < r.a) != (t == 0)) { i = min(i + end - x, r.units) - 1; continue; }      // the other half's
                const int b = n & 1;
                const bool sees = !idle && (reader < 0 || (reader >= lo && reader <= hi));      // any row of this warp
                if (!(ok = wait(&s_full[2 * t + b], (uint32_t)(n >> 1 & 1), 77))) break;
                tc5::fence_after();
                uint32_t pk[32];
                if (!sees) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) pk[e] = 0u;
                } else {
                    uint32_t sr[64];
                    tc5::ld32(S_t + lane_off + (uint32_t)(b * 64), sr);
                    tc5::ld32(S_t + lane_off + (uint32_t)(b * 64) + 32, sr + 32);
                    tc5::wait_ld();
                    const bool here = reader < 0 || member == reader;
                    if (reader >= 0) {
                        // keys that a row does not see become minus infinity (the scale is positive)
                        const int last = here ? table->pos[r.first + reader] - (x - before(r, reader)) * PAGE : -1;
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (c > last) sr[c] = 0xff800000u;
                    }
                    // P = 2^(score scale - maximum in use) as bfloat16 pairs; returns the sum of the page's P
                    auto exponentials = [&]() -> float {
                        const float mu = m_used == -INFINITY ? 0.f : m_used;
                        const unsigned long long sc2 = pack2(scale_log2, scale_log2), nmu2 = pack2(-mu, -mu);
                        unsigned long long l4[4] = {pack2(0.f, 0.f), pack2(0.f, 0.f), pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float x0, x1;
                            unpack2(fma2(pack2(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1])), sc2, nmu2), x0, x1);
                            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                            l4[e & 3] = add2(l4[e & 3], pack2(p0, p1));
                            pk[e] = pack_bf16(p0, p1);
                        }
                        float la, lb;
                        unpack2(add2(add2(l4[0], l4[1]), add2(l4[2], l4[3])), la, lb);
                        return la + lb;
                    };
                    // The maximum in use is that of the pages before (any is exact while nothing overflows): only where a row
                    // that sees the page has none yet, or the page's sum says that a score lies more than 2^64 above it, is the
                    // page's own found, O rescaled where it has grown by more than 2^8, and the page computed again.
                    float lpage = 0.f;
                    bool again = here && m_used == -INFINITY;
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
                            if (!fresh && __any_sync(0xffffffffu, had)) {
                                // P V of the page before must be complete before O is rescaled (that of this page waits for
                                // this warp's p_ready, that of two pages ago came before these scores: the phase is the one meant)
                                if (!(ok = wait(&pv_done[t], (uint32_t)((n - 1) & 1), 78))) break;
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
                }
                if (!idle) {
                    // P over this thread's own row of the scores it has read: nothing else uses this buffer now (the P V of
                    // two pages ago was issued before these scores, and the tensor core works in order)
                    tc5::st32(S_t + lane_off + (uint32_t)(b * 64), pk);
                    tc5::wait_st();
                }
                tc5::fence_before();
                __syncwarp();
                if (lane == 0) tma::mbar_arrive(&p_ready[2 * t + b]);
                ++n;
                fresh = false;
            }
            // The run's last P V (on a barrier of its own: by pv_done's parity, two phases not yet complete would look like the last
            // one being so), then the part of every row that has seen a page of the run
            if (!ok || !(ok = wait(&o_done[t], (uint32_t)(runs & 1), 79))) break;
            ++runs;
            tc5::fence_after();
            if (idle) continue;
            const bool seen = row < rows && (r.unit0 < r.prefix || max(r.unit0, r.prefix + before(r, member)) <
                                                                       min(r.unit0 + r.units, r.prefix + before(r, member + 1)));
            if (!__any_sync(0xffffffffu, seen)) continue;
            const size_t at = r.row0 + (size_t)blockIdx.x * ROWS + (size_t)member * G + row % G;
            float* dst = args.part_o + at * dv;
#pragma unroll 1
            for (int c0 = 0; c0 < (EXACT ? DV : dv); c0 += 32) {
                uint32_t o[32];
                tc5::ld32(O_t + lane_off + c0, o);
                tc5::wait_ld();
                if (seen) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8)
                        if (EXACT || c0 + c < dv) store8(dst + c0 + c, o + c);
                }
            }
            if (seen) args.part_ml[at] = make_float2(m_used, l);
            tc5::fence_before();
        }
    }
    pdl_wait();
    tc5::fence_before();
    __syncthreads();
    if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }       // let copies in flight land before the CTA goes away
        __syncthreads();
    }
    if (warp == 9) {
        tc5::fence_after();
        tc5::dealloc(tmem, TMEM_COLS);
    }
}

// A warp a row: its parts in the order of their runs, eight asked for at a time.
__global__ void __launch_bounds__(256) attn_shared_join_kernel(bf16* __restrict__ out, const int* __restrict__ seq_of_token, int ntok, int nq,
                                                               int nkv, const float* __restrict__ sink, float out_scale, const AttnShape sh,
                                                               const SharedArgs args) {
    pdl_launch();
    const int lane = threadIdx.x & 31, G = nq / nkv, dv = sh.dv, row = (int)blockIdx.x * 8 + (threadIdx.x >> 5);
    const bool in = row < ntok * nq;
    const int tok = in ? row / nq : 0, h = row - tok * nq, c = 4 * lane;
    const bool real = in && seq_of_token[tok] >= 0;
    pdl_wait();
    if (!in) return;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (real) {
        const int4 w = args.where[tok * nkv + h / G];
        const int np = w.z, first_own = w.w & 0xffff, n = np + (w.w >> 16);
        const size_t base = (size_t)w.x + h % G;
        for (int k0 = 0; k0 < n; k0 += 8) {
            float2 ml[8];
            float4 v[8];
            float top = M;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                ml[k] = make_float2(-INFINITY, 0.f);
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + k < n) {
                    const int run = k0 + k < np ? w.y + k0 + k : first_own + k0 + k - np;
                    const size_t at = base + (size_t)run * ROWS;
                    ml[k] = args.part_ml[at];
                    if (c < dv) v[k] = *reinterpret_cast<const float4*>(args.part_o + at * dv + c);
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
            if (top == -INFINITY) continue;
            const float f0 = fast_exp2(M - top);
            M = top;
            L *= f0; acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float f = fast_exp2(ml[k].x - top);
                L = fmaf(ml[k].y, f, L);
                acc.x = fmaf(v[k].x, f, acc.x); acc.y = fmaf(v[k].y, f, acc.y); acc.z = fmaf(v[k].z, f, acc.z); acc.w = fmaf(v[k].w, f, acc.w);
            }
        }
    }
    if (c >= dv) return;
    L = attn_sink_sum(L, M, sink, h);
    const float inv = L > 0.f ? out_scale / L : 0.f;
    const float y0 = attn_gate(acc.x * inv, sh, tok, h * dv + c), y1 = attn_gate(acc.y * inv, sh, tok, h * dv + c + 1);
    const float y2 = attn_gate(acc.z * inv, sh, tok, h * dv + c + 2), y3 = attn_gate(acc.w * inv, sh, tok, h * dv + c + 3);
    *reinterpret_cast<uint2*>(out + ((size_t)tok * nq + h) * dv + c) = make_uint2(pack_bf16(y0, y1), pack_bf16(y2, y3));
}

template <int DK, int DV, bool EXACT>
int launch_shared(const CUtensorMap& tk, const CUtensorMap& tv, const void* q, const int* positions, const int* seq_of_token,
                  const int* page_table, int max_pages, int nq, int nkv, float scale_log2, int n_pages, int* status, int d, int dv,
                  const SharedArgs& args, cudaStream_t stream) {
    // Q of two halves (boxes of 64 columns: 16 KB), the ring of K and V, barriers, the table
    constexpr int smem = 2 * (DK / 64) * 16384 + 128 * 1024 / ((DK + DV) / 64 * 8192) * ((DK + DV) / 64 * 8192) + 512 + (int)sizeof(Table);
    static int known[GG_MAX_DEVICES];
    auto kern = attn_shared_kernel<DK, DV, EXACT>;
    int resident = 0;
    const int rc = gg_resident(kern, THREADS, smem, known, resident);
    if (rc != 0) return rc;
    return gg_launch(kern, dim3(CTAS), dim3(THREADS), smem, stream, 1, tk, tv, (const bf16*)q, positions, seq_of_token, page_table, max_pages,
                     nq, nkv, scale_log2, n_pages, status, d, dv, args);
}

}  // namespace

// Decode attention (see gg_attn_decode_tma) of a step with shared prefixes: plan as at SharedArgs (at most 1,024 token rows);
// part: scratch of (nq ntok + 256 * 148) (dv + 2) + 4 ntok nkv floats, on a 32-byte boundary.
// status: codes 71-79 name the wait that ran out.
GG_API gg_attn_decode_shared(const void* q, const void* k_pool, const void* v_pool, void* out, const int* positions,
                             const int* seq_of_token, const int* page_table, int max_pages, int page_size, int n_pages, const int* plan,
                             int ntok, int nq, int nkv, int d, int dv, float scale, const float* sink, float out_scale, const void* gate,
                             long long ldg, float* part, long long part_floats, int* status, cudaStream_t stream) {
    if (ntok <= 0) return 0;
    if (page_size != PAGE || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > 16 || !attn_shape_ok(d, dv, 0, gate, ldg) || ntok > MAX_TOKENS ||
        n_pages <= 0 || max_pages <= 0 || status == nullptr || plan == nullptr)
        return GG_ERR_ARG;
    if ((((uintptr_t)q) & 15) || (((uintptr_t)k_pool) & 15) || (((uintptr_t)v_pool) & 15) || (((uintptr_t)out) & 15) || (((uintptr_t)part) & 31))
        return GG_ERR_ARG;
    const long long rows = (long long)nq * ntok + (long long)ROWS * CTAS;
    if (part == nullptr || part_floats < rows * (dv + 2) + 4ll * ntok * nkv || rows > 0x7fffffffll) return GG_ERR_ARG;
    // (units, and the rows of the pools, are counted in 32 bits: a row lists at most max_pages pages)
    const unsigned long long pool_rows = (unsigned long long)n_pages * nkv * PAGE;
    if (pool_rows > 0x7fffffffull || (unsigned long long)ntok * max_pages * nkv > 0x7fffffffull) return GG_ERR_ARG;
    CUtensorMap tk, tv;
    int rc;
    if ((rc = tma::make_map_bf16(&tk, k_pool, pool_rows, d, d, PAGE)) != 0) return rc;
    if ((rc = tma::make_map_bf16(&tv, v_pool, pool_rows, dv, dv, PAGE)) != 0) return rc;
    const float scale_log2 = scale * 1.4426950408889634f;
    float* where = part + rows * dv;
    const SharedArgs args = {plan, ntok, part, reinterpret_cast<int4*>(where), reinterpret_cast<float2*>(where + 4ll * ntok * nkv)};
#define GG_SHARED(DK_, DV_, EX_)                                                                                                   \
    launch_shared<DK_, DV_, EX_>(tk, tv, q, positions, seq_of_token, page_table, max_pages, nq, nkv, scale_log2, n_pages, status, d, \
                                 dv, args, stream)
    if (d == 128 && dv == 128) rc = GG_SHARED(128, 128, true);
    else if (d == 64 && dv == 64) rc = GG_SHARED(64, 64, true);
    else if (d <= 64 && dv <= 64) rc = GG_SHARED(64, 64, false);
    else if (d <= 64) rc = GG_SHARED(64, 128, false);
    else if (dv <= 64) rc = GG_SHARED(128, 64, false);
    else rc = GG_SHARED(128, 128, false);
#undef GG_SHARED
    if (rc != 0) return rc;
    const AttnShape sh = {d, dv, 0, (const bf16*)gate, ldg};
    return gg_launch(attn_shared_join_kernel, dim3((ntok * nq + 7) / 8), dim3(256), 0, stream, 1, (bf16*)out, seq_of_token, ntok, nq, nkv, sink,
                     out_scale, sh, args);
}

// 1 if this library was built with checked page tables (the debug build), else 0.
GG_API gg_attention_shared_checked() { return gg_debug_bounds(); }
