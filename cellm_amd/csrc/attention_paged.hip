// Attention over paged K/V whose pages many query rows share (gfx950): 8-bit pages for
// decode and prompts, and 8-bit or f16 pages for trees of drafted tokens.
//
//   s_p = scale * (q . k_p), capped: s = cap * tanh(s / cap)
//   o   = sum_p e^(s_p - M) v_p / sum_p e^(s_p - M),   M = max_p s_p
// over the positions p that the row sees: up to its own, the last `window` of them; or
// (trees) the context and, behind it, the drafted slots whose bit its mask has.  A missing
// page counts as zero keys and values.  8-bit keys and values are c * s with one scale per
// (token, kv head), which leaves both sums: q . k = s_k (q . c_k), and s_v joins the weight.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"

#pragma clang fp contract(off)

namespace cellm {

namespace {

constexpr int kThreads = 256;

// What a row sees: positions start..ctx - 1, then (masks) those of ctx..end - 1 whose bit is set.
struct Sight {
    int start, ctx, end;
    const uint64_t* bits;
    __device__ __forceinline__ bool sees(int p) const
    {
        return p >= start && (p < ctx || (p < end && (bits[(p - ctx) >> 6] >> ((p - ctx) & 63) & 1)));
    }
};

// false: the row has no position, or its mask no node, and its output is left as it was
__device__ __forceinline__ bool sight_of(const PagedAttnArgs& a, int row, Sight& s)
{
    const int cap = a.g.max_blocks * a.g.tpb;
    if (!a.masks) {
        const int p = a.pos[row];
        s.end = s.ctx = min(p, cap - 1) + 1;
        s.start = a.window > 0 ? max(s.ctx - a.window, 0) : 0;
        s.bits = nullptr;
        return p >= 0;
    }
    const int c = a.pos[row / a.per];
    int nodes = 0;
    s.bits = a.masks + (size_t)row * a.words;
    for (int w = 0; w < a.words; ++w) {
        const int left = a.per - 64 * w;
        const uint64_t m = left >= 64 ? ~0ull : (1ull << left) - 1;
        nodes += __popcll(s.bits[w] & m);
    }
    s.ctx = min(c, cap);
    s.end = min(s.ctx + a.per, cap);
    // the node stands at position ctx + nodes - 1 (its ancestors and itself)
    s.start = a.window > 0 ? max(s.ctx + nodes - a.window, 0) : 0;
    return c >= 0 && nodes > 0;
}

// element offset of head kvh's vector of position p, or -1 where its page is missing; and its number
template <bool Q8, int HD>
__device__ __forceinline__ long long vector_at(const KvGeom& g, int table, int p, int kvh)
{
    const int b = p / g.tpb;
    const uint32_t blk = g.bt[(size_t)table * g.max_blocks + b];
    if (blk >= (uint32_t)g.total_blocks) return -1;
    const long long page = (long long)blk * g.n_layers + g.layer;
    if constexpr (Q8) return (page * g.n_kv + kvh) * g.tpb + (p - b * g.tpb);
    else return (page * g.tpb + (p - b * g.tpb)) * g.n_kv + kvh;
}

// One block per (row, query head): 256 positions at a time, a score per thread, then HD
// threads per position.
template <bool Q8, int HD>
__global__ __launch_bounds__(kThreads) void attn_paged_plain_kernel(const PagedAttnArgs a)
{
    __shared__ float qs[HD], ws[kThreads], red[kThreads];
    __shared__ long long vec[kThreads];
    const int row = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads, kvh = head / (a.n_heads / a.g.n_kv);
    const int t = threadIdx.x, table = row / a.per;
    Sight si;
    if (!sight_of(a, row, si)) return;  // the same for the whole block
    if (t < HD) qs[t] = a.q[((size_t)row * a.n_heads + head) * HD + t];
    __syncthreads();
    const auto score = [&](int p, long long v) {
        float d = 0.0f;
        if (v >= 0) {
            if constexpr (Q8) {
                const u4_t* src = reinterpret_cast<const u4_t*>(static_cast<const int8_t*>(a.kc) + v * HD);
                for (int i = 0; i < HD / 16; ++i) {
                    const u4_t w = src[i];
#pragma unroll
                    for (int j = 0; j < 16; ++j) d = d + qs[16 * i + j] * (float)(int8_t)(w[j >> 2] >> (8 * (j & 3)));
                }
                d = d * a.ks[v];
            } else {
                const u4_t* src = reinterpret_cast<const u4_t*>(static_cast<const uint16_t*>(a.kc) + v * HD);
                for (int i = 0; i < HD / 8; ++i) {
                    const h8_t w = __builtin_bit_cast(h8_t, src[i]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) d = d + qs[8 * i + j] * (float)w[j];
                }
            }
        }
        d = d * a.scale;
        return a.cap > 0.0f ? tanhf(d / a.cap) * a.cap : d;
    };
    const auto reduce = [&](float v, auto op) {
        __syncthreads();
        red[t] = v;
        __syncthreads();
        for (int o = kThreads / 2; o > 0; o >>= 1) {
            if (t < o) red[t] = op(red[t], red[t + o]);
            __syncthreads();
        }
        return red[0];
    };
    float m = -INFINITY;
    for (int p = si.start + t; p < si.end; p += kThreads)
        if (si.sees(p)) m = fmaxf(m, score(p, vector_at<Q8, HD>(a.g, table, p, kvh)));
    m = reduce(m, [](float x, float y) { return fmaxf(x, y); });
    constexpr int NP = kThreads / HD;
    const int d = t % HD;
    float l = 0.0f, o = 0.0f;
    for (int p0 = si.start; p0 < si.end; p0 += kThreads) {
        const int p = p0 + t;
        long long v = -1;
        float w = 0.0f;
        if (p < si.end && si.sees(p)) {
            v = vector_at<Q8, HD>(a.g, table, p, kvh);
            w = expf(score(p, v) - m);
            l = l + w;
            if constexpr (Q8) w = v >= 0 ? w * a.vs[v] : 0.0f;
        }
        __syncthreads();
        vec[t] = v;
        ws[t] = w;
        __syncthreads();
        for (int j = t / HD; j < min(kThreads, si.end - p0); j += NP) {
            if (vec[j] < 0) continue;
            if constexpr (Q8) o = o + ws[j] * (float)static_cast<const int8_t*>(a.vc)[vec[j] * HD + d];
            else o = o + ws[j] * (float)static_cast<const _Float16*>(a.vc)[vec[j] * HD + d];
        }
    }
    l = reduce(l, [](float x, float y) { return x + y; });
    __syncthreads();
    red[t] = o;
    __syncthreads();
    if (t < HD) {
        o = 0.0f;
        for (int j = 0; j < NP; ++j) o = o + red[j * HD + t];
        a.out[((size_t)row * a.n_heads + head) * HD + t] = l != 0.0f ? o / l : 0.0f;
    }
}

}  // namespace

hipError_t launch_attention_paged(const PagedAttnArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)a.rows * (unsigned)a.n_heads);
    const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, st, a); };
    const bool q8 = a.ks != nullptr;
    if (a.head_dim == 64) q8 ? go(attn_paged_plain_kernel<true, 64>) : go(attn_paged_plain_kernel<false, 64>);
    else if (a.head_dim == 128) q8 ? go(attn_paged_plain_kernel<true, 128>) : go(attn_paged_plain_kernel<false, 128>);
    else q8 ? go(attn_paged_plain_kernel<true, 256>) : go(attn_paged_plain_kernel<false, 256>);
    return hipGetLastError();
}

}  // namespace cellm
