// Decode attention of a step some of whose rows share a prefix: the prefix's keys and values are read once for all its readers,
// as the rows of one tensor-core product, and every row's own positions by the decode kernel that a step without prefixes uses
// (attention_common.cuh), which adds the prefix's parts at its end.  With s_j = scale q . k_j, a part over a run of positions is
//     m >= some s_j of the run,   l = sum e^(s_j - m),   O = sum e^(s_j - m) v_j
// and parts add up as O = sum e^(m_i - m) O_i, l alike, whatever the m_i are; the output is O / l.
//
// The prefix kernel: a tile is up to 128 rows, members of a group times the query heads of a kv head.  Per page of 64 keys
// S = Q K^T (tcgen05.mma 128 x 64 x 16) lands in tensor memory, four warps take a row per thread, leave P as bfloat16 where S was
// and O += P V accumulates in tensor memory, as in the prefill kernel (attention_fast.cu), without its masks: every reader sees
// every key of the prefix.  All (group, tile, kv head)s' pages are one line of work cut into equal runs, one per CTA, so that
// neither the number of readers nor that of kv heads leaves an SM without work, and the grid is the same for every plan: a
// captured step replays with other groups.
//
// (Both as one kernel, whose CTAs are of the two kinds: a CTA of a kernel that allocates tensor memory keeps others off its SM
// until it has done so, so that the rows' CTAs, which never do, ran one an SM instead of two.  A row's own pages as pages of the
// prefix's product, seen by its rows only: they took the tensor core as long as any page.)
#include "attention_common.cuh"

namespace {

constexpr int SHARED_RUNS = 296;      // two CTAs per SM

// 32 bytes, a whole sector, at a time
__device__ __forceinline__ void store8(float* dst, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <int DK, int DV, bool EXACT>
__global__ void __launch_bounds__(192, 2) shared_prefix_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const bf16* q, const int* __restrict__ page_table,
    const int* __restrict__ seq_of_token, int max_pages, int nq, int nkv, float scale_log2, int n_pages, int* __restrict__ status,
    int d_, int dv_, const AttnShared shared) {
    constexpr int HK = DK / 64, HV = DV / 64;
    const int d = EXACT ? DK : d_, dv = EXACT ? DV : dv_, G = nq / nkv;
    constexpr int QBOX = SHARED_ROWS * 64 * 2;             // [64 columns x 128 rows] of Q: 16 KB
    constexpr int KBOX = 64 * 64 * 2;               // [64 columns x 64 keys] of K or V: 8 KB
    constexpr int Q_BYTES = HK * QBOX, K_STAGE = HK * KBOX, V_STAGE = HV * KBOX;
    constexpr int TMEM_COLS = 256;                  // two score buffers of 64 columns, then O
    // (the dynamic segment is the only shared memory and is asked to start on a 1024-byte boundary: two CTAs share an SM)
    extern __shared__ __align__(1024) uint8_t smem[];
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

    pdl_launch();                                   // (the whole grid is resident at once: the rule in common.cuh)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run = (int)blockIdx.x;
    const SharedPlan plan(shared);
    int total;
    plan.find(-1, -1, nkv, G, lane, total);
    const int per = plan.per(total, shared.runs), u_begin = min(run * per, total), u_end = min(u_begin + per, total);
    if (u_begin >= u_end) {                         // (every kernel of a step waits for the one before it: common.cuh)
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
    if (!ok && threadIdx.x == 0) atomicCAS(status, 0, 29);

    // The run is cut where the (tile, kv head) changes.  Every role walks the same cuts.
    struct Piece { int first, members, head, page0, pages, lead; size_t row0; };
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
        r.row0 = (size_t)nkv * G * r.first + (size_t)r.head * G * r.members + (size_t)run * SHARED_ROWS;
        return r;
    };
    // (a warp goes on or leaves as a whole: what follows a wait is for whole warps)
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) -> bool {
        return __all_sync(0xffffffffu, tma::mbar_wait(bar, phase, abort_flag, status, code));
    };

    int j = 0;                                      // pages so far
    if (warp == 4) {
        // The prefix's pages were written by earlier steps (this step's tokens go to pages of the rows' own), so they are
        // streamed before the kernel before this one has finished.
        for (int u = u_begin; u < u_end;) {
            const Piece r = piece_at(u);
            u += r.pages;
            if (lane == 0 && ok) {
                const int* pt = page_table + (size_t)seq_of_token[r.lead] * max_pages;
                for (int i = 0; i < r.pages; ++i, ++j) {
                    const int s = j & 1;
                    const uint32_t ph = (uint32_t)((j >> 1) & 1) ^ 1u;
                    const int row = (gg_page(pt, r.page0 + i, max_pages, PageBounds{n_pages, status}, 54) * nkv + r.head) * PAGE;
                    if (!(ok = tma::mbar_wait(&k_empty[s], ph, abort_flag, status, 71))) break;
                    tma::mbar_expect_tx(&k_full[s], K_STAGE);
#pragma unroll
                    for (int hf = 0; hf < HK; ++hf) tma::load_2d(Ks + s * K_STAGE + hf * KBOX, &tmK, &k_full[s], hf * 64, row);
                    if (!(ok = tma::mbar_wait(&v_empty[s], ph, abort_flag, status, 72))) break;
                    tma::mbar_expect_tx(&v_full[s], V_STAGE);
#pragma unroll
                    for (int hf = 0; hf < HV; ++hf) tma::load_2d(Vs + s * V_STAGE + hf * KBOX, &tmV, &v_full[s], hf * 64, row);
                }
            }
            __syncwarp();
        }
    } else if (warp == 5) {
        const uint32_t idesc_qk = tc5::idesc_bf16(SHARED_ROWS, 64, 0), idesc_pv = tc5::idesc_bf16(SHARED_ROWS, EXACT ? DV : (dv + 15) & ~15, 1);
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
            const bf16* src = q + ((size_t)plan.rows[r.first + member] * nq + (size_t)r.head * G + (row - member * G)) * d;
            if (pieces == 0) pdl_wait();                       // q, and the scratch is free
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
                float* dst = shared.part_o + (r.row0 + row) * dv;
#pragma unroll 1
                for (int c0 = 0; c0 < (EXACT ? DV : dv); c0 += 32) {
                    uint32_t o[32];
                    tc5::ld32(O_t + lane_off + c0, o);
                    tc5::wait_ld();
                    if (live) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            if (EXACT || c0 + c < dv) store8(dst + c0 + c, o + c);
                    }
                }
                if (live) shared.part_ml[r.row0 + row] = make_float2(m_used, l);
                tc5::fence_before();
            }
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
    if (warp == 5) {
        tc5::fence_after();
        tc5::dealloc(S_t, TMEM_COLS);
    }
}

template <int DK, int DV, bool EXACT>
int launch_prefix(const CUtensorMap& tk, const CUtensorMap& tv, const void* q, const int* page_table, const int* seq_of_token, int max_pages,
                  int nq, int nkv, float scale_log2, int n_pages, int* status, int d, int dv, const AttnShared& shared, cudaStream_t stream) {
    // Q, K x 2, V x 2 (boxes of 64 columns: 16 KB of Q, 8 KB of K or V), barriers
    constexpr int smem = (DK / 64) * (16384 + 2 * 8192) + (DV / 64) * 2 * 8192 + 256;
    static int known[GG_MAX_DEVICES];
    auto kern = shared_prefix_kernel<DK, DV, EXACT>;
    int resident = 0;
    const int rc = gg_resident(kern, 192, smem, known, resident);
    if (rc != 0) return rc;
    return gg_launch(kern, dim3(shared.runs), dim3(192), smem, stream, 1, tk, tv, (const bf16*)q, page_table, seq_of_token, max_pages, nq,
                     nkv, scale_log2, n_pages, status, d, dv, shared);
}

template <int DK, int DV, int STAGES, bool EXACT>
int launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const void* q, void* out, const int* positions, const int* seq_of_token,
                const int* page_table, int max_pages, int ntok, int nq, int nkv, float scale_log2, int splits, const float* sink,
                float out_scale, int n_pages, int* status, const AttnShape& sh, const AttnShared& shared, cudaStream_t stream) {
    constexpr int smem = decode_tma_smem<DK, DV, STAGES>(9);
    static int known[GG_MAX_DEVICES];
    auto kern = attn_decode_tma_kernel<DK, DV, STAGES, EXACT, true>;
    int resident = 0;
    const int rc = gg_resident(kern, 160, smem, known, resident);
    if (rc != 0) return rc;
    const long long ctas = (long long)ntok * nkv * splits;
    return gg_launch(kern, dim3(ntok, nkv, splits), dim3(160), smem, stream, splits, tk, tv, (const bf16*)q, (bf16*)out, (float*)nullptr,
                     (float*)nullptr, positions, seq_of_token, page_table, max_pages, nq, nkv, scale_log2, 0, splits, splits > 1 ? 1 : 0,
                     ctas <= resident ? 1 : 0, sink, out_scale, n_pages, status, sh, shared);
}

long long part_rows(int ntok, int nq) { return (long long)nq * ntok + (long long)SHARED_ROWS * SHARED_RUNS; }

}  // namespace

// Decode attention (see gg_attn_decode_tma) of a step with shared prefixes: plan as at AttnShared, part: scratch of
// (nq ntok + 128 * 296) (dv + 2) floats, on a 32-byte boundary.  splits: 1, 2, 4 or 8 CTAs share a row's own pages.
// status: codes 71-79 name the prefix kernel's wait that ran out, 11 and 12 the other's.
GG_API gg_attn_decode_shared(const void* q, const void* k_pool, const void* v_pool, void* out, const int* positions,
                             const int* seq_of_token, const int* page_table, int max_pages, int page_size, int n_pages, const int* plan,
                             int ntok, int nq, int nkv, int d, int dv, float scale, int splits, const float* sink, float out_scale,
                             const void* gate, long long ldg, float* part, long long part_floats, int* status, cudaStream_t stream) {
    if (ntok <= 0) return 0;
    if (page_size != PAGE || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > 16 || !attn_shape_ok(d, dv, 0, gate, ldg) || nkv > 65535 ||
        n_pages <= 0 || status == nullptr || plan == nullptr || !(splits == 1 || splits == 2 || splits == 4 || splits == 8))
        return GG_ERR_ARG;
    if ((((uintptr_t)q) & 15) || (((uintptr_t)k_pool) & 15) || (((uintptr_t)v_pool) & 15) || (((uintptr_t)part) & 31)) return GG_ERR_ARG;
    const long long rows = part_rows(ntok, nq);
    if (part == nullptr || part_floats < rows * (dv + 2) || rows > 0x7fffffffll) return GG_ERR_ARG;
    CUtensorMap tk, tv;
    int rc;
    const unsigned long long pool_rows = (unsigned long long)n_pages * nkv * PAGE;
    if (pool_rows > 0x7fffffffull) return GG_ERR_ARG;
    if ((rc = tma::make_map_bf16(&tk, k_pool, pool_rows, d, d, PAGE)) != 0) return rc;
    if ((rc = tma::make_map_bf16(&tv, v_pool, pool_rows, dv, dv, PAGE)) != 0) return rc;
    const float scale_log2 = scale * 1.4426950408889634f;
    const AttnShape sh = {d, dv, 0, (const bf16*)gate, ldg};
    const AttnShared shared = {plan, ntok, SHARED_RUNS, part, reinterpret_cast<float2*>(part + rows * dv)};
#define GG_PREFIX(DK_, DV_, EX_) \
    launch_prefix<DK_, DV_, EX_>(tk, tv, q, page_table, seq_of_token, max_pages, nq, nkv, scale_log2, n_pages, status, d, dv, shared, stream)
#define GG_ROWS(DK_, DV_, ST_, EX_)                                                                                                      \
    launch_rows<DK_, DV_, ST_, EX_>(tk, tv, q, out, positions, seq_of_token, page_table, max_pages, ntok, nq, nkv, scale_log2, splits, sink, \
                                    out_scale, n_pages, status, sh, shared, stream)
    if (d == 128 && dv == 128) return (rc = GG_PREFIX(128, 128, true)) != 0 ? rc : GG_ROWS(128, 128, 3, true);
    if (d == 64 && dv == 64) return (rc = GG_PREFIX(64, 64, true)) != 0 ? rc : GG_ROWS(64, 64, 4, true);
    if (d <= 64 && dv <= 64) return (rc = GG_PREFIX(64, 64, false)) != 0 ? rc : GG_ROWS(64, 64, 4, false);
    if (d <= 64) return (rc = GG_PREFIX(64, 128, false)) != 0 ? rc : GG_ROWS(64, 128, 4, false);
    if (dv <= 64) return (rc = GG_PREFIX(128, 64, false)) != 0 ? rc : GG_ROWS(128, 64, 4, false);
    return (rc = GG_PREFIX(128, 128, false)) != 0 ? rc : GG_ROWS(128, 128, 3, false);
#undef GG_PREFIX
#undef GG_ROWS
}

// 1 if this library was built with checked page tables (the debug build), else 0.
GG_API gg_attention_shared_checked() { return gg_debug_bounds(); }
