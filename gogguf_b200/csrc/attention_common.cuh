// What the bfloat16 attention kernels over the paged cache share (attention_fast.cu, attention_shared.cu): fragments,
// packed arithmetic, the sizes they take, and decode attention with the cache streamed by TMA, which either reads all of a
// row's positions or those behind a prefix that another kernel has been over for all its readers.
#pragma once
#include "tma_util.cuh"

namespace {

constexpr int PAGE = 64;

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Pairs of float32 in one 64-bit register for the packed arithmetic of sm_100 (two results per issue slot).
__device__ __forceinline__ unsigned long long pack2(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ void st_dsmem_f32(uint32_t local_addr, uint32_t rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

__device__ __forceinline__ float ld_dsmem_f32(uint32_t local_addr, uint32_t rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}

// from the shared memory of CTA `rank` of the cluster, at the address that `local` is in this CTA
__device__ __forceinline__ void attn_remote(uint32_t local, int rank, float& a, float& b) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(a), "=f"(b) : "r"(remote) : "memory");
}
__device__ __forceinline__ float4 attn_remote4(uint32_t local, int rank) {
    uint32_t remote;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
    return v;
}

__device__ __forceinline__ uint4 ldg16(const bf16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(smem);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm_x4(uint32_t* r, const void* p) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t* r, const void* p) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}

// element (row, 16-byte chunk) of a [rows][D] bf16 tile with the chunk index XOR-swizzled by the row
template <int D> __device__ __forceinline__ bf16* sw(bf16* tile, int row, int chunk) {
    return tile + row * D + ((chunk ^ (row & 7)) << 3);
}

// A softmax sink: a number per query head that joins the denominator as exp(sink[h]) (no key, no value, not
// scaled).  `l` is the sum of 2^(score - m) over the keys with m the maximum in use (in log2 units, -inf when no
// key was seen); what comes back is the denominator with the sink's share.
__device__ __forceinline__ float attn_sink_sum(float l, float m, const float* __restrict__ sink, int head) {
    if (sink == nullptr || m == -INFINITY) return l;
    return l + fast_exp2(sink[head] * 1.4426950408889634f - m);
}

// What the kernels below take beside one head size of 64 or 128: the key and value heads' own sizes d and dv (multiples
// of 8, at most the templates' DK and DV: what lies beyond them in a tile is zeros), chunks of positions (a position sees
// its own chunk only, counted from the sequence's start; 0: none), and a gate per output element (the result is
// multiplied by sigmoid(gate[token, head dv + i]); null: none).  EXACT kernels are those with d = DK and dv = DV.
struct AttnShape {
    int d, dv, chunk;
    const bf16* gate;
    long long ldg;
};
__device__ __forceinline__ float attn_gate(float v, const AttnShape& sh, int tok, int col) {
    if (sh.gate == nullptr) return v;
    return v / (1.0f + __expf(-__bfloat162float(sh.gate[(size_t)tok * sh.ldg + col])));
}
// the first position that a query at position p reads
__device__ __forceinline__ int attn_first(int p, int window, int chunk) {
    int lo = 0;
    if (window > 0 && p - window + 1 > 0) lo = p - window + 1;
    if (chunk > 0) lo = max(lo, p / chunk * chunk);
    return lo;
}

// ------------------------------------------------------------------------------------------- decode, TMA ring
// The same work as attn_decode_kernel with the cache streamed by TMA: one producer thread keeps a
// ring of whole pages (64 keys: K and V, [64 x 64]-column boxes, 128-byte swizzle) in flight, four
// consumer warps take 16 keys of each page, read fragments with ldmatrix and keep their own running
// maximum, sum and output; they are merged at the end as in the other kernel.  The copy engine
// decouples the loads from the arithmetic, which a warp that loads and computes in turn cannot.
// Largest cluster of splits: 8 is what every device takes; 16 needs the non-portable opt-in, which the
// launcher asks for once and falls back from (attn_max_cluster).
constexpr int MAX_ATT_CLUSTER = 16;

// What the other CTAs of a cluster push into this one (beyond the ring, so that they need not wait for it): their
// partial outputs for the slices of 32 this CTA merges, [rank][round][32], and their (max, sum) per query head.
constexpr int ATT_PUSH_MAX_OUT = 1024;                               // G * D up to which the splits are pushed
constexpr int ATT_RECV_O = (ATT_PUSH_MAX_OUT + 32 * 16) * 4;         // bytes: rank * rounds * 32 <= G * D + 32 * cs
constexpr int ATT_RECV_ML = 16 * 16 * 2 * 4;
constexpr int ATT_RECV_BYTES = ATT_RECV_O + ATT_RECV_ML;


// A prefix that several rows of a decode step read (attention_shared.cu).  The plan, integers of a step with room for `cap` token
// rows: how many groups; from word 4 on, per group the place of its first member in `rows` (and one place beyond the last
// group's), its pages and its first member; `rows`, the members' token rows group by group; per token row the pages that are its
// prefix (0: none), its group (-1: none) and its place among the group's members.  A group's members are cut into tiles of equal
// size whose rows, members times the query heads of a kv head, fit 128; the units of work are the pages of (group, tile, kv head)
// in that order, and run c, a CTA of the prefix kernel, takes `per` of them from c per on.  What a run leaves of a (tile, kv
// head) is a part: per row the values' sum, the maximum it was taken against and the sum of the weights.  The part's rows begin at
// row0 + 128 c, with row0 the rows of all (tile, kv head)s before: later parts are later in c or in row0, and 128 is the most a
// part has, so no two overlap.
struct AttnShared {
    const int* plan;
    int cap;                          // token rows that the plan has room for
    int runs;                         // CTAs of the prefix kernel
    float* part_o;                    // [rows][dv]
    float2* part_ml;                  // [rows] (maximum in log2 units, sum)
};
constexpr int SHARED_ROWS = 128;      // of a tile

struct SharedPlan {
    const int *count, *first, *pages, *lead, *rows, *pages_of, *group_of, *member_of;
    int cap;
    __device__ __forceinline__ SharedPlan(const AttnShared& a)
        : count(a.plan), first(a.plan + 4), pages(first + a.cap + 1), lead(pages + a.cap), rows(lead + a.cap), pages_of(rows + a.cap),
          group_of(pages_of + a.cap), member_of(group_of + a.cap), cap(a.cap) {}
    static __device__ __forceinline__ int tiles(int members, int G) {
        const int most = SHARED_ROWS / G;
        return (members + most - 1) / most;
    }
    // members of each tile but the last
    static __device__ __forceinline__ int tile_members(int members, int G) {
        const int n = tiles(members, G);
        return (members + n - 1) / n;
    }
    // units of a run: as many for each, and two at least (a part costs as much to write and to add as a page to read)
    static __device__ __forceinline__ int per(int total, int runs) { return max(2, (total + runs - 1) / runs); }

    // All units, and the group that unit u is of (u < 0: group `which`), by a whole warp: a lane a group.
    struct Group { int before, pages, first, members, lead; };
    __device__ __forceinline__ Group find(int u, int which, int nkv, int G, int lane, int& total) const {
        Group found = {};
        int groups = 1;
        total = 0;
        for (int g0 = 0; g0 < groups; g0 += 32) {
            const int g = min(g0 + lane, cap - 1);
            // (asked for before the number of groups is known: beyond the last one stands something that is not used)
            const int pg = pages[g], f = first[g], m = first[g + 1] - f, head = lead[g];
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
    // where the parts of a token row and kv head are (the first one's first row, and their number), by a whole warp
    __device__ __forceinline__ int2 where(int tok, int kvh, int nkv, int G, int runs, int lane) const {
        const int which = group_of[tok], mine = member_of[tok];
        if (which < 0) return make_int2(0, 0);
        int total;
        const Group g = find(-1, which, nkv, G, lane, total);
        const int tm = tile_members(g.members, G), p = per(total, runs), tile = mine / tm;
        const int u0 = g.before + (tile * nkv + kvh) * g.pages, c0 = u0 / p, c1 = (u0 + g.pages - 1) / p;
        return make_int2(nkv * G * (g.first + tile * tm) + kvh * G * min(tm, g.members - tile * tm) + c0 * SHARED_ROWS + (mine - tile * tm) * G,
                         c1 - c0 + 1);
    }
};

// The parts of one token row and kv head: `count` of them, 128 rows apart.
struct SharedParts {
    const float* o;
    const float2* ml;
    int count;
    __device__ __forceinline__ SharedParts(const AttnShared& a, int2 w, int dv) : o(a.part_o + (size_t)w.x * dv), ml(a.part_ml + w.x), count(w.y) {}
    // One warp's share of the parts (every `step`-th from k0 on) of the kv head's G rows, added up into sm_o [G][DV] and sm_ml
    // [G][2], four columns a lane; eight rows of parts are asked for at a time, whichever row or part they are of.
    template <int DV>
    __device__ __forceinline__ void add_up(int k0, int step, int G, int dv, int lane, float* sm_o, float* sm_ml) const {
        const int mine = k0 < count ? (count - 1 - k0) / step + 1 : 0;
        const bool in = lane * 4 < dv;
        if (mine == 0) {
            if (lane < G) { sm_ml[lane * 2] = -INFINITY; sm_ml[lane * 2 + 1] = 0.f; }
            for (int r = 0; in && r < G; ++r) *reinterpret_cast<float4*>(sm_o + r * DV + lane * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
            return;
        }
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        int r_ask = 0, i_ask = 0, r = 0, i = 0;          // row and part that are asked for, and that are added, next
        while (r < G) {
            float2 v[8];
            float4 x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = make_float2(-INFINITY, 0.f);
                x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r_ask < G) {
                    const size_t at = (size_t)(k0 + i_ask * step) * SHARED_ROWS + r_ask;
                    v[e] = ml[at];
                    if (in) x[e] = *reinterpret_cast<const float4*>(o + at * dv + lane * 4);
                    if (++i_ask == mine) { i_ask = 0; ++r_ask; }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (r >= G) break;
                const float top = fmaxf(M, v[e].x);
                if (top != -INFINITY) {
                    const float f = fast_exp2(M - top), w = fast_exp2(v[e].x - top);
                    M = top;
                    L = fmaf(v[e].y, w, L * f);
                    acc.x = fmaf(x[e].x, w, acc.x * f); acc.y = fmaf(x[e].y, w, acc.y * f);
                    acc.z = fmaf(x[e].z, w, acc.z * f); acc.w = fmaf(x[e].w, w, acc.w * f);
                }
                if (++i == mine) {
                    if (in) *reinterpret_cast<float4*>(sm_o + r * DV + lane * 4) = acc;
                    if (lane == 0) { sm_ml[r * 2] = M; sm_ml[r * 2 + 1] = L; }
                    i = 0; ++r;
                    M = -INFINITY; L = 0.f;
                    acc = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
        }
    }
};

// SHARED: a row's first pages are those of its group's prefix, whose parts the kernel before has left; this one reads the
// others and adds the parts.
template <int DK, int DV, int STAGES, bool EXACT, bool SHARED>
__global__ void __launch_bounds__(160) attn_decode_tma_kernel(
    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const bf16* q, bf16* __restrict__ out, float* __restrict__ part_o, float* __restrict__ part_ml,
    const int* __restrict__ positions, const int* __restrict__ seq_of_token,
    const int* __restrict__ page_table, int max_pages, int nq, int nkv, float scale_log2, int window, int nsplit,
    int cluster_reduce, int early_release, const float* __restrict__ sink, float out_scale, int n_pages,
    int* __restrict__ status, const AttnShape sh, const AttnShared shared) {
    // A grid that is resident as a whole lets the next kernel's CTAs in at once: they share the SMs' free
    // shared memory and start fetching weights.  A grid of several waves releases only after its pages (the
    // rule on dependent launches in common.cuh): until then its own waiting CTAs should get the SMs.
    if (early_release) pdl_launch();
    constexpr int HK = DK / 64, HV = DV / 64;
    constexpr int BOX_BYTES = 64 * 64 * 2;                 // 8 KB
    constexpr int STAGE_BYTES = (HK + HV) * BOX_BYTES;     // K halves then V halves
    constexpr int KS = DK / 16, NT = DV / 8;
    const int d = EXACT ? DK : sh.d, dv = EXACT ? DV : sh.dv;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + STAGES * STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    volatile int* abort_flag = (volatile int*)(empty + STAGES);
    int2* parts_at = (int2*)(empty + STAGES + 1);                                     // (SHARED) where the prefix's parts are
    float* recv_o = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES + 256);      // see ATT_RECV_BYTES
    float* recv_ml = recv_o + ATT_RECV_O / 4;

    const int tok = blockIdx.x, kvh = blockIdx.y, split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int G = nq / nkv;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { tma::mbar_init(&full[s], 1); tma::mbar_init(&empty[s], 4); }
        *abort_flag = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&tmK);
        tma::prefetch_map(&tmV);
    }
    __syncthreads();
    // The step's integer inputs (positions, sequence rows, page tables) were copied to the device before the
    // step's first kernel started.  Of the cache, the kernels of this step write only position `pos` (one new
    // token per sequence), which lies in page pos / 64; every earlier page was written by earlier steps.  So
    // the producer starts streaming those pages while the projection before this kernel is still finishing,
    // and waits for it only before the page that holds the new token; the consumers wait before they read q.
    const int b = seq_of_token[tok];
    const int pos = b >= 0 ? positions[tok] : -1;
    const int prefix = SHARED ? SharedPlan(shared).pages_of[tok] : 0;

    int lo = 0, p_begin = 0, p_end = 0;
    if (b >= 0) {
        lo = attn_first(pos, window, sh.chunk);
        int first = lo / PAGE;
        const int last = pos / PAGE;
        if constexpr (SHARED) {
            first = max(first, prefix);
        }
        const int pps = (last - first + 1 + nsplit - 1) / nsplit;
        p_begin = first + split * pps;
        p_end = min(last + 1, p_begin + pps);
    }
    const int npg = max(0, p_end - p_begin);

    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f; }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    if (warp == 4) {
        if (lane == 0) {
            const int* pt = page_table + (size_t)b * max_pages;
            const int newest = pos / PAGE;
            bool waited = false;
            for (int i = 0; i < npg; ++i) {
                const int s = i % STAGES;
                const uint32_t ph = (uint32_t)(i / STAGES) & 1u;
                if (!waited && p_begin + i >= newest) { pdl_wait(); waited = true; }
                if (!tma::mbar_wait(&empty[s], ph ^ 1u, abort_flag, status, 11)) break;
                tma::mbar_expect_tx(&full[s], STAGE_BYTES);
                const int row = (gg_page(pt, p_begin + i, max_pages, PageBounds{n_pages, status}, 44) * nkv + kvh) * PAGE;
                uint8_t* dst = smem + s * STAGE_BYTES;
#pragma unroll
                for (int hf = 0; hf < HK; ++hf) tma::load_2d(dst + hf * BOX_BYTES, &tmK, &full[s], hf * 64, row);
#pragma unroll
                for (int hf = 0; hf < HV; ++hf) tma::load_2d(dst + (HK + hf) * BOX_BYTES, &tmV, &full[s], hf * 64, row);
            }
        }
        if constexpr (SHARED) {
            // (while the others work on the pages)
            __syncwarp();
            const int2 w = SharedPlan(shared).where(tok, kvh, nkv, G, shared.runs, lane);
            if (lane == 0) *parts_at = w;
        }
    } else if (npg > 0) {
        // Q fragments in the standard A layout: row = head of the group, k = head dimension
        uint32_t qa[KS][4];
        pdl_wait();
        {
            const bf16* q0 = q + ((size_t)tok * nq + (size_t)kvh * G) * d;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int c = ks * 16 + 2 * t;
                const bool in0 = EXACT || c < d, in1 = EXACT || c + 8 < d;
                qa[ks][0] = g < G && in0 ? *reinterpret_cast<const uint32_t*>(q0 + (size_t)g * d + c) : 0u;
                qa[ks][1] = g + 8 < G && in0 ? *reinterpret_cast<const uint32_t*>(q0 + (size_t)(g + 8) * d + c) : 0u;
                qa[ks][2] = g < G && in1 ? *reinterpret_cast<const uint32_t*>(q0 + (size_t)g * d + c + 8) : 0u;
                qa[ks][3] = g + 8 < G && in1 ? *reinterpret_cast<const uint32_t*>(q0 + (size_t)(g + 8) * d + c + 8) : 0u;
            }
        }
        const int krow = warp * 16;     // this warp's 16 keys of every page
        for (int i = 0; i < npg; ++i) {
            const int s = i % STAGES;
            const uint32_t ph = (uint32_t)(i / STAGES) & 1u;
            if (!tma::mbar_wait(&full[s], ph, abort_flag, status, 12)) break;
            const uint8_t* st = smem + s * STAGE_BYTES;
            const int key0 = (p_begin + i) * PAGE + krow;
            float sc[2][4];
            sc[0][0] = sc[0][1] = sc[0][2] = sc[0][3] = 0.f;
            sc[1][0] = sc[1][1] = sc[1][2] = sc[1][3] = 0.f;
            if (key0 <= pos && key0 + 15 >= lo) {      // whole-warp decision: any visible key among these 16?
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bf16* box = reinterpret_cast<const bf16*>(st + (ks >> 2) * BOX_BYTES);
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
                        const int kidx = key0 + j * 8 + 2 * t + (e & 1);
                        const float v = (kidx >= lo && kidx <= pos) ? sc[j][e] * scale_log2 : -INFINITY;
                        sc[j][e] = v;
                        mx[e >> 1] = fmaxf(mx[e >> 1], v);
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
                    const bf16* box = reinterpret_cast<const bf16*>(st + (HK + (np >> 2)) * BOX_BYTES);
                    uint32_t vb[4];
                    ldsm_x4_trans(vb, sw<64>(const_cast<bf16*>(box), krow + (lane & 7) + (((lane >> 3) & 1) << 3), (np & 3) * 2 + (lane >> 4)));
                    mma16816(o[2 * np], pa, vb[0], vb[1]);
                    mma16816(o[2 * np + 1], pa, vb[2], vb[3]);
                }
            }
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&empty[s]);
        }
    }
    pdl_wait();               // (returns at once where it was already called) the output buffer is free from here
    if (!early_release) pdl_launch();
    __syncthreads();          // all pages consumed (or the CTA gave up): the ring can be reused for the merge
    if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }       // let copies in flight land before the CTA goes away
        __syncthreads();
    }
    // what this CTA adds up: the four warps' shares of its pages, and (SHARED) the five warps' shares of the prefix's parts,
    // which go round the CTAs of a row
    constexpr int ADDENDS = SHARED ? 9 : 4;
    float* sm_o = reinterpret_cast<float*>(smem);                 // [ADDENDS][16][DV]
    float* sm_ml = sm_o + ADDENDS * 16 * DV;                      // [ADDENDS][16][2]
    float* res_o = sm_ml + ADDENDS * 16 * 2;                      // [16][DV]  this CTA's merged output (cluster form)
    float* res_ml = res_o + 16 * DV;                              // [16][2]
    if (warp < 4) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        // only the G rows that are query heads go on (the MMA tile has 16)
        if (g < G) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
                *reinterpret_cast<float2*>(&sm_o[(warp * 16 + g) * DV + n * 8 + 2 * t]) = make_float2(o[n][0], o[n][1]);
            if (t == 0) { sm_ml[(warp * 16 + g) * 2] = m[0]; sm_ml[(warp * 16 + g) * 2 + 1] = l[0]; }
        }
        if (g + 8 < G) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
                *reinterpret_cast<float2*>(&sm_o[(warp * 16 + g + 8) * DV + n * 8 + 2 * t]) = make_float2(o[n][2], o[n][3]);
            if (t == 0) { sm_ml[(warp * 16 + g + 8) * 2] = m[1]; sm_ml[(warp * 16 + g + 8) * 2 + 1] = l[1]; }
        }
    }
    if constexpr (SHARED)
        SharedParts(shared, *parts_at, dv).add_up<DV>(split * 5 + warp, 5 * nsplit, G, dv, lane, sm_o + (4 + warp) * 16 * DV, sm_ml + (4 + warp) * 16 * 2);
    __syncthreads();
    for (int idx = threadIdx.x; idx < G * dv; idx += blockDim.x) {
        const int r = idx / dv, c = idx - r * dv;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < ADDENDS; ++w) M = fmaxf(M, sm_ml[(w * 16 + r) * 2]);
        float L = 0.f, acc = 0.f;
        if (M != -INFINITY) {
#pragma unroll
            for (int w = 0; w < ADDENDS; ++w) {
                const float f = fast_exp2(sm_ml[(w * 16 + r) * 2] - M);
                L += sm_ml[(w * 16 + r) * 2 + 1] * f;
                acc += sm_o[(w * 16 + r) * DV + c] * f;
            }
        }
        const int head = kvh * G + r;
        if (nsplit == 1) {
            const float Ls = attn_sink_sum(L, M, sink, head);
            out[((size_t)tok * nq + head) * dv + c] =
                __float2bfloat16_rn(attn_gate(Ls > 0.f ? acc * out_scale / Ls : 0.f, sh, tok, head * dv + c));
        } else if (cluster_reduce && G * dv <= ATT_PUSH_MAX_OUT) {
            // straight into the shared memory of the CTA that merges this output (slices of 32 go round the
            // ranks), and this head's (max, sum) to every CTA: no load has to cross the cluster afterwards
            const int chunk = idx >> 5, owner = chunk % nsplit, round = chunk / nsplit;
            const int rounds = ((G * dv + 31) / 32 + nsplit - 1) / nsplit;
            st_dsmem_f32(tma::smem_u32(recv_o + (split * rounds + round) * 32 + (idx & 31)), (uint32_t)owner, acc);
            if (c == 0) {
                for (int k = 0; k < nsplit; ++k) {
                    st_dsmem_f32(tma::smem_u32(recv_ml + (split * 16 + r) * 2), (uint32_t)k, M);
                    st_dsmem_f32(tma::smem_u32(recv_ml + (split * 16 + r) * 2 + 1), (uint32_t)k, L);
                }
            }
        } else if (cluster_reduce) {
            res_o[r * dv + c] = acc;
            if (c == 0) { res_ml[r * 2] = M; res_ml[r * 2 + 1] = L; }
        } else {
            const size_t pi = ((size_t)tok * nq + head) * nsplit + split;
            part_o[pi * dv + c] = acc;
            if (c == 0) { part_ml[pi * 2] = M; part_ml[pi * 2 + 1] = L; }
        }
    }
    if (cluster_reduce && G * dv <= ATT_PUSH_MAX_OUT) {
        // The splits of one (token, kv head) form a cluster; what the ranks pushed is complete after one barrier,
        // and every CTA merges its slice of the G x D outputs, in rank order, from its own shared memory.
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const int rounds = ((G * dv + 31) / 32 + nsplit - 1) / nsplit;
        for (int round = warp; round < rounds; round += 5) {
            const int idx = (round * nsplit + split) * 32 + lane;
            if (idx >= G * dv) continue;
            const int r = idx / dv;
            float M = -INFINITY;
            for (int k = 0; k < nsplit; ++k) M = fmaxf(M, recv_ml[(k * 16 + r) * 2]);
            float L = 0.f, acc = 0.f;
            if (M != -INFINITY) {
                for (int k = 0; k < nsplit; ++k) {
                    const float f = fast_exp2(recv_ml[(k * 16 + r) * 2] - M);
                    L += recv_ml[(k * 16 + r) * 2 + 1] * f;
                    acc += recv_o[(k * rounds + round) * 32 + lane] * f;
                }
            }
            const float Ls = attn_sink_sum(L, M, sink, kvh * G + r);
            out[((size_t)tok * nq + kvh * G) * dv + idx] =
                __float2bfloat16_rn(attn_gate(Ls > 0.f ? acc * out_scale / Ls : 0.f, sh, tok, kvh * G * dv + idx));
        }
    } else if (cluster_reduce) {
        // (more than 1,024 outputs per kv head do not fit the receive area: the owner pulls instead)
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const uint32_t ro = tma::smem_u32(res_o), rm = tma::smem_u32(res_ml);
        for (int idx = split * blockDim.x + threadIdx.x; idx < G * dv; idx += nsplit * blockDim.x) {
            const int r = idx / dv, c = idx - r * dv;
            float ms[MAX_ATT_CLUSTER], ls[MAX_ATT_CLUSTER], as[MAX_ATT_CLUSTER];
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < MAX_ATT_CLUSTER; ++k) {
                if (k < nsplit) {
                    ms[k] = ld_dsmem_f32(rm + 4u * (r * 2), k);
                    ls[k] = ld_dsmem_f32(rm + 4u * (r * 2 + 1), k);
                    as[k] = ld_dsmem_f32(ro + 4u * idx, k);
                } else { ms[k] = -INFINITY; ls[k] = 0.f; as[k] = 0.f; }
                M = fmaxf(M, ms[k]);
            }
            float L = 0.f, acc = 0.f;
            if (M != -INFINITY) {
#pragma unroll
                for (int k = 0; k < MAX_ATT_CLUSTER; ++k) {
                    const float f = fast_exp2(ms[k] - M);
                    L += ls[k] * f;
                    acc += as[k] * f;
                }
            }
            const float Ls = attn_sink_sum(L, M, sink, kvh * G + r);
            out[((size_t)tok * nq + kvh * G + r) * dv + c] =
                __float2bfloat16_rn(attn_gate(Ls > 0.f ? acc * out_scale / Ls : 0.f, sh, tok, (kvh * G + r) * dv + c));
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <int DK, int DV, int STAGES>
constexpr int decode_tma_smem(int addends = 4) {
    constexpr int ring = STAGES * ((DK + DV) / 64) * 8192;    // bytes: a box of 8 KB per 64 columns of K and of V
    const int merge = ((addends + 1) * 16 * DV + (addends + 1) * 16 * 2) * 4;
    return (ring > merge ? ring : merge) + 1024 + 256 + ATT_RECV_BYTES;
}

// The sizes the kernels here take: d and dv multiples of 8 up to 128, the exact kernels where both are 64 or both
// 128.  A gate's rows start on 16-byte boundaries.
static bool attn_shape_ok(int d, int dv, int chunk, const void* gate, long long ldg) {
    if (d <= 0 || dv <= 0 || d > 128 || dv > 128 || (d & 7) || (dv & 7) || chunk < 0) return false;
    return gate == nullptr || ((((uintptr_t)gate) & 15) == 0 && (ldg & 7) == 0);
}
// call F<DK, DV, EXACT>(...) for the sizes
#define GG_ATTN_SIZES(F, ...)                                                              \
    do {                                                                                   \
        if (d == 128 && dv == 128) return F<128, 128, true>(__VA_ARGS__);                  \
        if (d == 64 && dv == 64) return F<64, 64, true>(__VA_ARGS__);                      \
        if (d <= 64 && dv <= 64) return F<64, 64, false>(__VA_ARGS__);                     \
        if (d <= 64) return F<64, 128, false>(__VA_ARGS__);                                \
        if (dv <= 64) return F<128, 64, false>(__VA_ARGS__);                               \
        return F<128, 128, false>(__VA_ARGS__);                                            \
    } while (0)

}  // namespace
