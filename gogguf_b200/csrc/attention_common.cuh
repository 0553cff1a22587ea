// What the bfloat16 attention kernels over the paged cache share (attention_fast.cu, attention_shared.cu): fragments, packed
// arithmetic, a cluster's shared memory, sinks, gates, and the sizes they take.
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

__device__ __forceinline__ uint4 ldg16(const bf16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

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
// The sizes the kernels take: d and dv multiples of 8 up to 128, the exact kernels where both are 64 or both
// 128.  A gate's rows start on 16-byte boundaries.
static bool attn_shape_ok(int d, int dv, int chunk, const void* gate, long long ldg) {
    if (d <= 0 || dv <= 0 || d > 128 || dv > 128 || (d & 7) || (dv & 7) || chunk < 0) return false;
    return gate == nullptr || ((((uintptr_t)gate) & 15) == 0 && (ldg & 7) == 0);
}

}  // namespace
