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

template <bool IN_PLACE>
__global__ void __launch_bounds__(THREADS) shape_logits_kernel(const float* logits, long long ld, float* out, long long ldo, int V,
                                                               const int* __restrict__ ring_rows, int rings, const Shaping s) {
    __shared__ int count[SLICE];
    __shared__ int bias_at[SLICE];
    const int r = blockIdx.y, lo = blockIdx.x * SLICE, n = min(SLICE, V - lo);
    pdl_launch();
    const bool sparse = s.hist != nullptr || s.bias_start != nullptr;
    if (sparse) {
        for (int i = threadIdx.x; i < SLICE; i += THREADS) { count[i] = 0; bias_at[i] = 0; }
        __syncthreads();
    }
    pdl_wait();
    const int ring = ring_rows != nullptr ? ring_rows[r] : r;
    const bool known = ring >= 0 && ring < rings;
    const float* x = logits + (size_t)r * ld + lo;
    float* y = out + (size_t)r * ldo + lo;
    if (sparse) {
        if (known && s.hist != nullptr) {
            const int* h = s.hist + (size_t)ring * s.last_n;
            const int m = min(s.hist_len[ring], s.last_n);
            for (int t = threadIdx.x; t < m; t += THREADS) {
                const int id = h[t];
                if (id >= lo && id - lo < n) atomicAdd(&count[id - lo], 1);
            }
        }
        if (known && s.bias_start != nullptr) {
            const int e = min(s.bias_start[ring + 1], s.biases);
            for (int t = max(s.bias_start[ring], 0) + threadIdx.x; t < e; t += THREADS) {
                const int id = s.bias_ids[t];
                if (id >= lo && id - lo < n) atomicMax(&bias_at[id - lo], t + 1);     // of an id that is listed twice, the last entry
            }
        }
        __syncthreads();
    }
    const int state = known && s.masks != nullptr ? s.mask_rows[ring] : -1;
    // (a state beyond the table allows nothing)
    const int* bits = state >= 0 && state < s.states ? s.masks + (size_t)state * s.words : nullptr;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const int v = lo + i;
        const bool allowed = state < 0 || (bits != nullptr && (bits[v >> 5] >> (v & 31) & 1));
        if (!allowed) { y[i] = -INFINITY; continue; }
        const int c = sparse ? count[i] : 0, b = sparse ? bias_at[i] : 0;
        if (IN_PLACE && c == 0 && b == 0) continue;
        y[i] = shaped(x[i], c, b, s);
    }
}

}  // namespace

// out[r] = the shaped logits[r] for R rows of V; out == logits (and ldo == ld): in place, where only what changes is touched.
// ring_rows (null: row r's request is r) names each row's request among `rings`.
GG_API gg_shape_logits(const float* logits, long long ld, float* out, long long ldo, int R, int V, const int* ring_rows, int rings,
                       const int* hist, const int* hist_len, int last_n, float repeat, float frequency, float presence,
                       const int* bias_start, const int* bias_ids, const float* bias_values, int biases, const int* masks,
                       const int* mask_rows, int states, int words, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (V <= 0 || ld < V || ldo < V || R > 65535 || rings <= 0 || !(repeat > 0.f)) return GG_ERR_ARG;
    if (hist != nullptr && (hist_len == nullptr || last_n <= 0)) return GG_ERR_ARG;
    if (bias_start != nullptr && (bias_ids == nullptr || bias_values == nullptr || biases < 0)) return GG_ERR_ARG;
    if (masks != nullptr && (mask_rows == nullptr || states <= 0 || words < (V + 31) / 32)) return GG_ERR_ARG;
    const Shaping s = {hist, hist_len, last_n, repeat, frequency, presence, bias_start, bias_ids, bias_values, biases,
                       masks, mask_rows, states, words};
    const dim3 grid((V + SLICE - 1) / SLICE, R);
    if (out == logits) {
        if (ld != ldo) return GG_ERR_ARG;
        if (hist == nullptr && bias_start == nullptr && masks == nullptr) return 0;
        return gg_launch(shape_logits_kernel<true>, grid, dim3(THREADS), 0, stream, 1, logits, ld, out, ldo, V, ring_rows, rings, s);
    }
    return gg_launch(shape_logits_kernel<false>, grid, dim3(THREADS), 0, stream, 1, logits, ld, out, ldo, V, ring_rows, rings, s);
}
