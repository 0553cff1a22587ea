// Shaping of a step's logits before a token is drawn from them, and what a drawn token changes.
//
// Row r, id v, c = how often v stands among the last ids of the row's request:
//     z = x[v];   if c > 0:  z = z > 0 ? z / repeat : z * repeat,  z -= frequency c + presence
//     z += bias of v;   ids that the request's grammar state does not allow: z = -inf
// (the repeat penalty as in the reference, pkg/sampler/penalties.go:5-32, which has neither of the others).
//
// The rows are cut into slices, one block each: it counts those of the request's last ids that lie in its slice in shared
// memory (whole numbers, so that the order of the additions does not matter), notes the biases that do, and passes once over
// its logits.  Whatever the number of ids, no id is compared with another.
#include <climits>
#include <cstring>

#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int SLICE = 4096;                 // logits per block
constexpr int PER = SLICE / THREADS;

struct Shaping {
    const int* hist;                        // [rings, last_n] ids, hist_len of them in use; null: no penalties
    const int* hist_len;
    int last_n;
    float repeat, frequency, presence;
    const int* bias_start;                  // [rings + 1]; null: no biases
    const int* bias_ids;
    const float* bias_values;
    int biases;
    const int* masks;                       // [states, words] bits of allowed ids; null: no grammar
    const int* mask_rows;                   // [rings] state of a request, negative: none
    int states, words;
};

__device__ __forceinline__ float shaped(float x, int c, int b, const Shaping& s) {
    if (c > 0) {
        if (s.repeat != 1.0f) x = x > 0.f ? x / s.repeat : x * s.repeat;
        x -= fmaf(s.frequency, (float)c, s.presence);
    }
    if (b > 0) x += s.bias_values[b - 1];
    return x;
}

// VEC: logits of a load (4: rows on 16-byte boundaries).  A thread's logits lie THREADS * VEC apart, so that a warp's lie side by
// side.  A slice is 4 us of waiting for loads that depend on one another (the row's request, its numbers, its ids and its state's
// bits) around 32 KB of traffic, so what does not depend is asked for together, the logits first, and as many CTAs as fit an SM
// share it: of a logit's word the lower half counts its id, the upper one is its bias's place in the request's list, plus one
// (WIDE: two words, for windows or lists beyond 65,535).
template <bool IN_PLACE, int VEC, bool WIDE>
__global__ void __launch_bounds__(THREADS, 6) shape_logits_kernel(const float* logits, long long ld, float* out, long long ldo, int V,
                                                               const int* __restrict__ ring_rows, int rings, const Shaping s) {
    constexpr int GROUPS = PER / VEC;
    __shared__ __align__(16) unsigned seen[WIDE ? 2 : 1][SLICE];
    const int r = blockIdx.y, lo = blockIdx.x * SLICE, n = min(SLICE, V - lo);
    pdl_launch();
    const bool sparse = s.hist != nullptr || s.bias_start != nullptr;
    if (sparse) {
        for (int i = threadIdx.x * 4; i < (WIDE ? 2 : 1) * SLICE; i += THREADS * 4) *reinterpret_cast<uint4*>(seen[0] + i) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    }
    pdl_wait();
    const float* x = logits + (size_t)r * ld + lo;
    float* y = out + (size_t)r * ldo + lo;
    float v[GROUPS][VEC];
    if (!IN_PLACE) {
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
            const int i = (k * THREADS + threadIdx.x) * VEC;
            if (VEC == 4 && i + 4 <= n) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i));
                v[k][0] = f.x; v[k][1 % VEC] = f.y; v[k][2 % VEC] = f.z; v[k][3 % VEC] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[k][e] = i + e < n ? __ldcs(x + i + e) : 0.f;
            }
        }
    }
    const int ring = ring_rows != nullptr ? ring_rows[r] : r;
    const bool known = ring >= 0 && ring < rings;
    const int ids = known && s.hist != nullptr ? min(s.hist_len[ring], s.last_n) : 0;
    const int state = known && s.masks != nullptr ? s.mask_rows[ring] : -1;
    // (a start beyond the list is a list that is over: what is added to it below stays within 32 bits)
    const int b0 = known && s.bias_start != nullptr ? min(max(s.bias_start[ring], 0), s.biases) : 0;
    const int b1 = known && s.bias_start != nullptr ? min(s.bias_start[ring + 1], s.biases) : 0;
    const int* h = s.hist + (size_t)ring * s.last_n;
    int first_id = -1, first_bias = -1;
    if ((int)threadIdx.x < ids) first_id = h[threadIdx.x];
    if (b0 + (int)threadIdx.x < b1) first_bias = s.bias_ids[b0 + threadIdx.x];
    // bits of allowed ids, a thread's groups'  (a state beyond the table allows nothing)
    unsigned allowed[GROUPS];
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        const int at = lo + (k * THREADS + threadIdx.x) * VEC;
        allowed[k] = state < 0 ? 0xffffffffu : state < s.states && at < V ? (unsigned)s.masks[(size_t)state * s.words + (at >> 5)] >> (at & 31) : 0u;
    }
    bool any = false;                               // an id of this slice is penalised or has a bias
    if (sparse) {
        auto count = [&](int id) {
            if (id >= lo && id - lo < n) { atomicAdd(&seen[0][id - lo], 1u); any = true; }
        };
        count(first_id);
        int t = threadIdx.x + THREADS;
        for (; t < ids; t += 4 * THREADS) {
            int some[4];                            // (asked for together)
#pragma unroll
            for (int k = 0; k < 4; ++k) some[k] = t + k * THREADS < ids ? h[t + k * THREADS] : -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) count(some[k]);
        }
        for (int e = b0 + threadIdx.x; e < b1; e += THREADS) {
            const int id = e < b0 + THREADS ? first_bias : s.bias_ids[e];
            if (id < lo || id - lo >= n) continue;
            any = true;
            // (of an id that is listed twice, the last entry)
            if (WIDE) {
                atomicMax(&seen[1][id - lo], (unsigned)(e - b0 + 1));
            } else {
                unsigned old = seen[0][id - lo], was;
                do {
                    was = old;
                    old = atomicCAS(&seen[0][id - lo], was, max(was >> 16, (unsigned)(e - b0 + 1)) << 16 | (was & 0xffffu));
                } while (old != was);
            }
        }
        any = __syncthreads_or(any);
    }
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        const int i = (k * THREADS + threadIdx.x) * VEC;
        if (i >= n) break;
        unsigned w[VEC] = {}, u[VEC] = {};
        bool some = false;                          // of this group is seen or has a bias
        if (any) {
            if (VEC == 4) {
                const uint4 w4 = *reinterpret_cast<const uint4*>(seen[0] + i);
                w[0] = w4.x; w[1 % VEC] = w4.y; w[2 % VEC] = w4.z; w[3 % VEC] = w4.w;
                if (WIDE) {
                    const uint4 u4 = *reinterpret_cast<const uint4*>(seen[WIDE ? 1 : 0] + i);
                    u[0] = u4.x; u[1 % VEC] = u4.y; u[2 % VEC] = u4.z; u[3 % VEC] = u4.w;
                }
            } else {
                w[0] = seen[0][i];
                if (WIDE) u[0] = seen[WIDE ? 1 : 0][i];
            }
            unsigned both = 0u;
#pragma unroll
            for (int e = 0; e < VEC; ++e) both |= w[e] | u[e];
            some = both != 0u;
        }
        auto one = [&](float z, int e) -> float {
            const int c = WIDE ? (int)w[e] : (int)(w[e] & 0xffffu), b = WIDE ? (int)u[e] : (int)(w[e] >> 16);
            return shaped(z, c, b > 0 ? b0 + b : 0, s);
        };
        if (IN_PLACE) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (i + e >= n) break;
                if (!(allowed[k] >> e & 1)) y[i + e] = -INFINITY;
                else if (some && (w[e] | u[e]) != 0u) y[i + e] = one(x[i + e], e);
            }
        } else {
            if (some) {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if ((w[e] | u[e]) != 0u) v[k][e] = one(v[k][e], e);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (!(allowed[k] >> e & 1)) v[k][e] = -INFINITY;
            if (VEC == 4 && i + 4 <= n) {
                __stcs(reinterpret_cast<float4*>(y + i), make_float4(v[k][0], v[k][1 % VEC], v[k][2 % VEC], v[k][3 % VEC]));
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (i + e < n) __stcs(y + i + e, v[k][e]);
            }
        }
    }
}

// What a drawn id changes for its request: the last ids, the grammar's state; an id that the state does not allow becomes -1.
__global__ void shape_advance_kernel(int* tokens, const int* __restrict__ ring_rows, int R, int rings, int* hist, int* hist_len, int* hist_pos,
                                     int last_n, int* states, const int* classes, const int* next, int n_states, int n_classes, int V) {
    pdl_launch();
    pdl_wait();
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= R) return;
    const int ring = ring_rows != nullptr ? ring_rows[r] : r;
    if (ring < 0 || ring >= rings) return;
    int id = tokens[r];
    if (states != nullptr && states[ring] >= 0) {
        const int s = states[ring];
        const int c = id >= 0 && id < V ? classes[id] : -1;
        const int to = s < n_states && c >= 0 && c < n_classes ? next[(size_t)s * n_classes + c] : -1;
        if (to < 0) tokens[r] = id = -1;
        else states[ring] = to;
    }
    if (hist != nullptr && id >= 0) {
        const int p = hist_pos[ring];
        hist[(size_t)ring * last_n + p] = id;
        hist_pos[ring] = p + 1 == last_n ? 0 : p + 1;
        if (hist_len[ring] < last_n) hist_len[ring] += 1;
    }
}

}  // namespace

// out[r] = the shaped logits[r] for R rows of V; out == logits (and ldo == ld): in place, where only what changes is touched.
// ring_rows (null: row r's request is r) names each row's request among `rings`.
//
// The arguments come packed, eight bytes each: of a call of 5 us on the device ctypes took 3.7 us of the host to convert 23 of them.
struct ShapeCall {
    const float* logits;
    long long ld;
    float* out;
    long long ldo, R, V;
    const int* ring_rows;
    long long rings;
    const int *hist, *hist_len;
    long long last_n;
    double repeat, frequency, presence;
    const int *bias_start, *bias_ids;
    const float* bias_values;
    long long biases;
    const int *masks, *mask_rows;
    long long states, words;
};
static_assert(sizeof(ShapeCall) == 22 * 8, "as the caller packs it");

GG_API gg_shape_logits(const void* call, cudaStream_t stream) {
    ShapeCall c;
    memcpy(&c, call, sizeof(c));
    if (c.R <= 0) return 0;
    if (c.V <= 0 || c.V > INT_MAX - SLICE || c.ld < c.V || c.ldo < c.V || c.R > 65535 || c.rings <= 0 || c.rings > INT_MAX || !(c.repeat > 0.)) return GG_ERR_ARG;
    if (c.hist != nullptr && (c.hist_len == nullptr || c.last_n <= 0 || c.last_n > INT_MAX - 4 * THREADS)) return GG_ERR_ARG;
    if (c.bias_start != nullptr && (c.bias_ids == nullptr || c.bias_values == nullptr || c.biases < 0 || c.biases > INT_MAX - THREADS)) return GG_ERR_ARG;
    if (c.masks != nullptr && (c.mask_rows == nullptr || c.states <= 0 || c.states > INT_MAX || c.words < (c.V + 31) / 32 || c.words > INT_MAX)) return GG_ERR_ARG;
    const Shaping s = {c.hist, c.hist_len, (int)c.last_n, (float)c.repeat, (float)c.frequency, (float)c.presence, c.bias_start, c.bias_ids,
                       c.bias_values, (int)c.biases, c.masks, c.mask_rows, (int)c.states, (int)c.words};
    const float* logits = c.logits;
    float* out = c.out;
    const long long ld = c.ld, ldo = c.ldo;
    const int R = (int)c.R, V = (int)c.V;
    const dim3 grid((V + SLICE - 1) / SLICE, R);
    const bool vec = ((uintptr_t)logits & 15) == 0 && ((uintptr_t)out & 15) == 0 && (R == 1 || ((ld | ldo) & 3) == 0);
    const bool in_place = out == logits;
    if (in_place && R > 1 && ld != ldo) return GG_ERR_ARG;
    if (in_place && s.hist == nullptr && s.bias_start == nullptr && s.masks == nullptr) return 0;
    // (a request's own list is no longer than all of them)
    const bool wide = (s.hist != nullptr && s.last_n > 65535) || s.biases > 65534;
#define GG_SHAPE(WIDE_) (in_place ? (vec ? shape_logits_kernel<true, 4, WIDE_> : shape_logits_kernel<true, 1, WIDE_>) \
                                  : (vec ? shape_logits_kernel<false, 4, WIDE_> : shape_logits_kernel<false, 1, WIDE_>))
    auto kern = wide ? GG_SHAPE(true) : GG_SHAPE(false);
#undef GG_SHAPE
    return gg_launch(kern, grid, dim3(THREADS), 0, stream, 1, logits, ld, out, ldo, V, c.ring_rows, (int)c.rings, s);
}

// R drawn ids (in place); the requests' last ids (hist null: none are kept) as gg_history_append appends to them; their grammar states
// (null: none; negative: that request has none) over `next` [n_states, n_classes] and a class per id.  A request stands in one row
// at most.
GG_API gg_shape_advance(int* tokens, const int* ring_rows, int R, int rings, int* hist, int* hist_len, int* hist_pos, int last_n, int* states,
                        const int* classes, const int* next, int n_states, int n_classes, int V, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (rings <= 0 || (hist != nullptr && (hist_len == nullptr || hist_pos == nullptr || last_n <= 0))) return GG_ERR_ARG;
    if (states != nullptr && (classes == nullptr || next == nullptr || n_states <= 0 || n_classes <= 0 || V <= 0)) return GG_ERR_ARG;
    return gg_launch(shape_advance_kernel, dim3((R + 127) / 128), dim3(128), 0, stream, 1, tokens, ring_rows, R, rings, hist, hist_len, hist_pos,
                     last_n, states, classes, next, n_states, n_classes, V);
}
