// Attention over 4-bit pages, one block per row and query head: a chunk of positions' scores, a
// thread each, then their weighted values, a dim each, with a running maximum and sum.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"
#include "kv_pages.hpp"

#pragma clang fp contract(off)

namespace cellm {

namespace {

constexpr int kThreads = 256;

template <int HD>
__device__ __forceinline__ void word_of(const void* codes, const void* scales, size_t vn, int i, float (&x)[8])
{
    const uint32_t w = static_cast<const uint32_t*>(codes)[vn * (HD / 8) + i];
    const uint32_t m = static_cast<const uint32_t*>(scales)[vn * (HD / 32) + i / 4];
    const h2_t s = as_h2((m & 0xFFFFu) * 0x10001u), z = as_h2((m >> 16) * 0x10001u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const h2_t v = values4(w >> (4 * j) & 0x000F000Fu, s, z);
        x[j] = (float)v[0];
        x[j + 4] = (float)v[1];
    }
}

template <int HD>
__global__ __launch_bounds__(kThreads) void attn_q4_kernel(const PagedAttnArgs a)
{
    __shared__ float w[kThreads];
    __shared__ long long vec[kThreads];
    __shared__ float red[kThreads];
    const int t = threadIdx.x, head = blockIdx.x, row = blockIdx.y + gridDim.y * blockIdx.z;
    if (row >= a.rows) return;
    int table = row / a.per;
    if (a.starts) {
        if (row >= a.starts[a.tables]) return;
        int lo = 0, hi = a.tables;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (a.starts[mid] <= row ? lo : hi) = mid;
        }
        table = lo;
    }
    if (a.pos[row] < 0) return;
    const int end = min(a.pos[row], a.g.max_blocks * a.g.tpb - 1) + 1, start = a.window > 0 ? max(end - a.window, 0) : 0;
    const int kvh = head / (a.n_heads / a.g.n_kv);
    const float* q = a.q + ((size_t)row * a.n_heads + head) * HD;
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
    float M = -INFINITY, L = 0.0f, o = 0.0f;
    bool nan = false;
    for (int p0 = start; p0 < end; p0 += kThreads) {
        const int p = p0 + t;
        float s = -INFINITY;
        long long vn = -1;
        if (p < end) {
            vn = vector_of(a.g, table, p);
            float d = 0.0f;
            if (vn >= 0) vn += (long long)kvh * a.g.tpb;
            for (int i = 0; i < HD / 8; ++i) {
                float x[8] = {};
                if (vn >= 0) word_of<HD>(a.kc, a.ks, (size_t)vn, i, x);
                for (int j = 0; j < 8; ++j) d += q[8 * i + j] * x[j];
            }
            s = d * a.scale;
            if (a.cap > 0.0f) s = tanhf(s / a.cap) * a.cap;
            nan |= s != s;
        }
        const float m = fmaxf(M, reduce(s, [](float x, float y) { return fmaxf(x, y); }));
        const float e = m > -INFINITY ? expf(s - m) : 0.0f, ratio = M > -INFINITY ? expf(M - m) : 0.0f;
        L = L * ratio + reduce(e, [](float x, float y) { return x + y; });
        w[t] = e;
        vec[t] = vn;
        __syncthreads();
        if (t < HD) {
            o *= ratio;
            for (int j = 0; j < min(kThreads, end - p0); ++j) {
                if (vec[j] < 0) continue;
                float x[8];
                word_of<HD>(a.vc, a.vs, (size_t)vec[j], t / 8, x);
                float v = 0.0f;
                for (int i = 0; i < 8; ++i) v = t % 8 == i ? x[i] : v;
                o += w[j] * v;
            }
        }
        M = m;
    }
    nan = __syncthreads_or(nan);
    if (t < HD) a.out[((size_t)row * a.n_heads + head) * HD + t] = nan ? __builtin_nanf("") : L != 0.0f ? o / L : 0.0f;
}

}  // namespace

hipError_t launch_attention_q4(const PagedAttnArgs& a, hipStream_t st)
{
    const unsigned y = (unsigned)std::min(a.rows, 32768);
    const dim3 grid((unsigned)a.n_heads, y, (unsigned)((a.rows + y - 1) / y));
    if (a.head_dim == 64) hipLaunchKernelGGL(attn_q4_kernel<64>, grid, dim3(kThreads), 0, st, a);
    else if (a.head_dim == 128) hipLaunchKernelGGL(attn_q4_kernel<128>, grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL(attn_q4_kernel<256>, grid, dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace cellm
