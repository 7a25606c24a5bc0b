// A serving step over a paged K/V cache whose lengths only the device knows (gfx950): pages and
// rows of the step from the sessions' lengths, q and k normed per head, rotated and written
// through the slot map to f16, 8-bit or 4-bit pages, and 4-bit pages read back.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"
#include "kv_pages.hpp"

#pragma clang fp contract(off)  // norm and RoPE: products and sums are rounded one by one

namespace cellm {

namespace {

constexpr int kThreads = 256;

// ---- the pages and rows of a step -----------------------------------------------------
// Session t holds ctx tokens in ceil(ctx / tpb) pages and asks for `add` more.  With running sums
// over the sessions, P of the pages that these need and R of their rows,
//   it gets them where P <= pages free and R <= rows: in order, up to the first that does not fit.
// Page i of those handed out (counted over the sessions) is entry count - 1 - i of the free
// list, after the pages of finished sessions (add < 0) have been put onto its end.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// inclusive sum over the block's threads; scan: kPlanWaves words
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* scan)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) scan[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += scan[w];
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(const KvPlanArgs a)
{
    __shared__ uint32_t scan[kPlanWaves];
    __shared__ uint32_t last[2];   // pages and rows of the last session that fits
    const int t = threadIdx.x, lane = t & 63;
    const auto pages_of = [&](long long tokens) { return (uint32_t)((tokens + a.tpb - 1) / a.tpb); };
    long long count = max(a.free_count[0], 0);
    if (count > a.free_capacity) count = a.free_capacity;

    // ---- finished sessions give their pages back, in the order of sessions and positions
    for (int t0 = 0; t0 < a.tables; t0 += kPlanThreads) {
        const int s = t0 + t;
        const int ctx = s < a.tables ? a.ctx[s] : -1, add = s < a.tables ? a.add[s] : 0;
        uint32_t entries = 0, valid = 0;
        if (ctx >= 0 && add < 0) entries = min(pages_of(ctx), (uint32_t)a.max_blocks);
        const auto each = [&](auto&& f) {  // the wave's finished sessions, 64 entries at a time
            for (unsigned long long todo = __ballot(entries > 0); todo; todo &= todo - 1) {
                const int src = __builtin_ctzll(todo);
                const uint32_t n = __shfl(entries, src);
                const uint32_t* row = a.bt + (size_t)(t0 + (t & ~63) + src) * a.max_blocks;
                for (uint32_t e0 = 0; e0 < n; e0 += 64) {
                    const uint32_t blk = e0 + lane < n ? row[e0 + lane] : ~0u;
                    f(src, blk, __ballot(blk < (uint32_t)a.total_blocks));
                }
            }
        };
        each([&](int src, uint32_t, unsigned long long there) {
            if (lane == src) valid += (uint32_t)__popcll(there);
        });
        const uint32_t up = block_scan(valid, scan);
        uint32_t at = up - valid;  // of the pages that this round gives back
        each([&](int src, uint32_t blk, unsigned long long there) {
            const uint32_t first = __shfl(at, src);
            const long long i = count + first + __popcll(there & ((1ull << lane) - 1));
            if (there >> lane & 1 && i < a.free_capacity) a.free_blocks[i] = blk;
            if (lane == src) at += (uint32_t)__popcll(there);
        });
        __syncthreads();
        if (t == kPlanThreads - 1) last[0] = up;
        __syncthreads();
        count = min(count + last[0], (long long)a.free_capacity);
    }
    __syncthreads();  // the free list as it is now

    // ---- sessions in order, up to the first whose pages or rows are not there
    long long pages0 = 0, rows0 = 0;  // of the sessions before this round's
    if (t == 0) a.starts[0] = 0;
    for (int t0 = 0; t0 < a.tables; t0 += kPlanThreads) {
        const int s = t0 + t;
        const int ctx = s < a.tables ? a.ctx[s] : -1, add = s < a.tables ? a.add[s] : 0;
        const bool valid = ctx >= 0 && add > 0 && (long long)ctx + add <= (long long)a.max_blocks * a.tpb;
        const uint32_t held = ctx > 0 ? pages_of(ctx) : 0;
        const uint32_t need = valid ? pages_of((long long)ctx + add) - held : 0;
        const uint32_t asked = valid ? (uint32_t)min(add, a.rows + 1) : 0;
        const uint32_t p = block_scan(need, scan), r = block_scan(asked, scan);
        const bool fits = pages0 + p <= count && rows0 + r <= a.rows;
        if (t < 2) last[t] = 0;
        __syncthreads();
        const unsigned long long in = __ballot(fits);
        if (in && lane == 63 - __builtin_clzll(in)) {  // sums rise with the sessions
            atomicMax(&last[0], p);
            atomicMax(&last[1], r);
        }
        __syncthreads();
        if (s < a.tables) {
            a.starts[s + 1] = (int32_t)(rows0 + (fits ? r : last[1]));
            a.lens_out[s] = fits && valid ? ctx + add : ctx >= 0 && add < 0 ? 0 : ctx;
        }
        if (fits && valid) {
            uint32_t* row = a.bt + (size_t)s * a.max_blocks + held;
            const uint32_t* top = a.free_blocks + (count - 1 - (pages0 + p - need));
            for (uint32_t j = 0; j < need; ++j) row[j] = top[-(long long)j];
        }
        const bool full = !__syncthreads_and(fits);
        pages0 += last[0];
        rows0 += last[1];
        if (full) {  // nothing more fits: the others wait
            for (int e = t0 + kPlanThreads + t; e < a.tables; e += kPlanThreads) {
                const int c = a.ctx[e];
                a.starts[e + 1] = (int32_t)rows0;
                a.lens_out[e] = c >= 0 && a.add[e] < 0 ? 0 : c;
            }
            break;
        }
        __syncthreads();
    }
    if (t == 0) a.free_out[0] = (int32_t)(count - pages0);
    __syncthreads();

    // ---- positions and slots of the rows
    for (int r = t; r < a.rows; r += kPlanThreads) {
        int pos = -1, slot = -1;
        if (r < rows0) {
            int lo = 0, hi = a.tables;  // starts[lo] <= r < starts[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                (a.starts[mid] <= r ? lo : hi) = mid;
            }
            pos = a.lens_out[lo] - (a.starts[lo + 1] - r);
            const int b = pos / a.tpb;
            const uint32_t blk = a.bt[(size_t)lo * a.max_blocks + b];
            if (blk < (uint32_t)a.total_blocks) slot = (int)(blk * (uint32_t)a.tpb) + (pos - b * a.tpb);
        }
        a.pos[r] = pos;
        a.slots[r] = slot;
    }
}

// ---- norm, rotation and write ---------------------------------------------------------
//   y = (x * inv) * w,  inv = f32(1 / sqrt(sum x^2 / HD + eps))
// for each head of q and k, the sum and the root in 64 bits, so that inv (and with it every bit of
// the result) does not hang on the order of the sum; then RoPE as in kv_cache.hip, and q to q_out,
// k and v to the row's slot.
__device__ __forceinline__ double lane_xor64(double v, int o)
{
    return __shfl_xor(v, o);
}

struct NormWriteArgs {
    NormRopeArgs n;
    int rows, n_heads;
    int units, tpb, layer, n_layers, n_kv;
    long long slots_end;
};

// One team of HD / 8 lanes per head vector: a row's query heads, then its K heads, then its V heads.  Lane l holds dims
// 4 l .. 4 l + 3 and HD / 2 + 4 l .. HD / 2 + 4 l + 3: the pairs of the rotate-half layout, two pairs of each run of
// the interleaved one, and 8 lanes hold two groups of 4-bit codes.
template <int HD, int FMT, int WDT>
__global__ __launch_bounds__(kThreads) void norm_rope_write_kernel(const NormWriteArgs A)
{
    constexpr int T = HD / 8, H = HD / 2;
    const NormRopeArgs& a = A.n;
    const int per_row = A.n_heads + 2 * A.n_kv, l = threadIdx.x % T;
    const uint32_t vec = blockIdx.x * (kThreads / T) + threadIdx.x / T;  // 32 bits: the host checks the count
    if (vec >= (uint32_t)A.rows * (uint32_t)per_row) return;              // whole teams
    const int r = (int)(vec / (uint32_t)per_row), h = (int)(vec - (uint32_t)r * (uint32_t)per_row);
    const bool is_q = h < A.n_heads, is_v = h >= A.n_heads + A.n_kv;
    const int kvh = is_q ? 0 : is_v ? h - A.n_heads - A.n_kv : h - A.n_heads;
    const int p = a.pos[r];
    if (p < 0) return;
    const int slot = a.slots[r];
    if (!is_q && (slot < 0 || slot >= A.slots_end)) return;
    const int e0 = 4 * l, e1 = H + 4 * l;
    const float* src = is_q ? a.q + ((size_t)r * A.n_heads + h) * HD
                            : (is_v ? a.v : a.k) + ((size_t)r * A.n_kv + kvh) * HD;
    const f4_t x0 = *reinterpret_cast<const f4_t*>(src + e0), x1 = *reinterpret_cast<const f4_t*>(src + e1);
    float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    const void* weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    if (weight) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += (double)x[i] * (double)x[i];
#pragma unroll
        for (int o = 1; o < T; o <<= 1) ss += lane_xor64(ss, o);
        const float inv = (float)(1.0 / sqrt(ss / HD + (double)a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = x[i] * inv;
            x[i] = y * load_f32<WDT>(weight, (i < 4 ? e0 : e1 - 4) + i);
        }
    }
    if (a.cos_sin && !is_v) {
        const float2* cs = reinterpret_cast<const float2*>(a.cos_sin) + (size_t)min(p, a.table_positions - 1) * H;
        const auto turn = [&](int u, int w, float2 c) {
            const float lo = x[u], hi = x[w];
            x[u] = lo * c.x - hi * c.y;
            x[w] = hi * c.x + lo * c.y;
        };
        if (!a.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) turn(i, 4 + i, cs[4 * l + i]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                turn(2 * i, 2 * i + 1, cs[2 * l + i]);
                turn(4 + 2 * i, 5 + 2 * i, cs[H / 2 + 2 * l + i]);
            }
        }
    }
    if (is_q) {
        float* dst = a.q_out + ((size_t)r * A.n_heads + h) * HD;
        *reinterpret_cast<f4_t*>(dst + e0) = f4_t{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f4_t*>(dst + e1) = f4_t{x[4], x[5], x[6], x[7]};
        return;
    }
    const int blk = slot / A.tpb, off = slot - blk * A.tpb;
    const size_t page = (size_t)blk * A.n_layers + A.layer;
    if constexpr (FMT == KV_F16) {
        uint16_t* dst = static_cast<uint16_t*>(is_v ? a.vc : a.kc) + ((page * A.tpb + off) * A.n_kv + kvh) * HD;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            asm("" : "+v"(x[2 * i]), "+v"(x[2 * i + 1]));  // the f32 products are what f16 rounds
            w[i] = as_u32(h2_t{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
        }
        *reinterpret_cast<u2_t*>(dst + e0) = u2_t{w[0], w[1]};
        *reinterpret_cast<u2_t*>(dst + e1) = u2_t{w[2], w[3]};
        return;
    }
    const size_t vn = (page * A.n_kv + kvh) * A.tpb + off;
    if constexpr (FMT == KV_Q8) {
        uint32_t w[2];
        const float s = quantise8<T>(x, w);
        int8_t* dst = static_cast<int8_t*>(is_v ? a.vc : a.kc) + vn * HD;
        *reinterpret_cast<uint32_t*>(dst + e0) = w[0];
        *reinterpret_cast<uint32_t*>(dst + e1) = w[1];
        if (l == 0) static_cast<float*>(is_v ? a.vs : a.ks)[vn] = s;
    }
    if constexpr (FMT == KV_Q4) {
        uint16_t* dst = static_cast<uint16_t*>(is_v ? a.vc : a.kc) + vn * (HD / 4);
        uint32_t* sc = static_cast<uint32_t*>(is_v ? a.vs : a.ks) + vn * (HD / 32);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float y[4] = {x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]};
            uint32_t s;
            dst[u * (H / 4) + l] = (uint16_t)quantise4(y, s);
            if (l % 8 == 0) sc[u * (H / 32) + l / 8] = s;
        }
    }
}

// ---- 4-bit pages read back --------------------------------------------------------------
// A word of codes per thread.
template <int HD, int DT>
__global__ __launch_bounds__(kThreads) void kv_read_q4_kernel(const uint32_t* __restrict__ kc, const uint32_t* __restrict__ ks,
                                                              const uint32_t* __restrict__ vc, const uint32_t* __restrict__ vs,
                                                              const int32_t* __restrict__ pos, int rows, int per, KvGeom g,
                                                              void* __restrict__ ko, void* __restrict__ vo)
{
    constexpr int T = HD / 8;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;  // 32 bits: the host checks the count
    if (i >= (uint32_t)rows * (uint32_t)g.n_kv * T) return;
    const uint32_t vec = i / T, row = vec / (uint32_t)g.n_kv;
    const int l = (int)(i % T), kvh = (int)(vec - row * (uint32_t)g.n_kv), r = (int)row;
    const int p = pos[r];
    if (p < 0) return;
    const long long v0 = vector_of(g, r / per, p);
    const size_t vn = v0 < 0 ? 0 : (size_t)v0 + (size_t)kvh * g.tpb;
    const auto one = [&](const uint32_t* c, const uint32_t* s, void* out) {
        const uint32_t w = v0 < 0 ? 0 : c[vn * T + l], m = v0 < 0 ? 0 : s[vn * (HD / 32) + l / 4];
        const h2_t sc = as_h2(both_low(m)), z = as_h2(both_high(m));
        _Float16 x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // nibbles j and j + 4
            const h2_t v = values4(w >> (4 * j) & 0x000F000Fu, sc, z);
            x[j] = v[0];
            x[j + 4] = v[1];
        }
        if constexpr (DT == DT_F32) {
            f4_t* o = reinterpret_cast<f4_t*>(out) + 2 * (size_t)i;
            o[0] = f4_t{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
            o[1] = f4_t{(float)x[4], (float)x[5], (float)x[6], (float)x[7]};
        } else {
            u4_t o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == DT_F16) o[j] = as_u32(h2_t{x[2 * j], x[2 * j + 1]});
                else o[j] = (uint32_t)bf16_rne((float)x[2 * j]) | (uint32_t)bf16_rne((float)x[2 * j + 1]) << 16;
            }
            reinterpret_cast<u4_t*>(out)[i] = o;
        }
    };
    one(kc, ks, ko);
    one(vc, vs, vo);
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t st)
{
    hipLaunchKernelGGL(kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_norm_rope_write(const NormRopeArgs& n, int rows, int n_heads, int head_dim, int fmt, const KvGeom& g,
                                  hipStream_t st)
{
    NormWriteArgs a{};
    a.n = n;
    a.rows = rows;
    a.n_heads = n_heads;
    a.tpb = g.tpb;
    a.layer = g.layer;
    a.n_layers = g.n_layers;
    a.n_kv = g.n_kv;
    a.slots_end = (long long)g.total_blocks * g.tpb;
    const long long vecs = (long long)rows * (n_heads + 2 * g.n_kv);
    const auto go = [&](auto hd, auto fm, auto wt) {
        constexpr int HD = decltype(hd)::value, V = kThreads / (HD / 8);
        hipLaunchKernelGGL((norm_rope_write_kernel<HD, decltype(fm)::value, decltype(wt)::value>),
                           dim3((unsigned)((vecs + V - 1) / V)), dim3(kThreads), 0, st, a);
    };
    const auto by_weight = [&](auto hd, auto fm) {
        if (n.weight_dtype == DT_F32) go(hd, fm, std::integral_constant<int, DT_F32>{});
        else if (n.weight_dtype == DT_F16) go(hd, fm, std::integral_constant<int, DT_F16>{});
        else go(hd, fm, std::integral_constant<int, DT_BF16>{});
    };
    const auto by_format = [&](auto hd) {
        if (fmt == KV_F16) by_weight(hd, std::integral_constant<int, KV_F16>{});
        else if (fmt == KV_Q8) by_weight(hd, std::integral_constant<int, KV_Q8>{});
        else by_weight(hd, std::integral_constant<int, KV_Q4>{});
    };
    if (head_dim == 64) by_format(std::integral_constant<int, 64>{});
    else if (head_dim == 128) by_format(std::integral_constant<int, 128>{});
    else by_format(std::integral_constant<int, 256>{});
    return hipGetLastError();
}

hipError_t launch_kv_read_q4(const void* kc, const void* ks, const void* vc, const void* vs, const int32_t* pos, int rows,
                             int per, int head_dim, const KvGeom& g, void* k_out, void* v_out, int out_dtype, hipStream_t st)
{
    const auto go = [&](auto hd, auto dt) {
        constexpr int HD = decltype(hd)::value, DT = decltype(dt)::value;
        const long long n = (long long)rows * g.n_kv * (HD / 8);
        const auto words = [](const void* p) { return static_cast<const uint32_t*>(p); };
        hipLaunchKernelGGL((kv_read_q4_kernel<HD, DT>), dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                           st, words(kc), words(ks), words(vc), words(vs), pos, rows, per, g, k_out, v_out);
    };
    const auto by_type = [&](auto hd) {
        if (out_dtype == DT_F32) go(hd, std::integral_constant<int, DT_F32>{});
        else if (out_dtype == DT_F16) go(hd, std::integral_constant<int, DT_F16>{});
        else go(hd, std::integral_constant<int, DT_BF16>{});
    };
    if (head_dim == 64) by_type(std::integral_constant<int, 64>{});
    else if (head_dim == 128) by_type(std::integral_constant<int, 128>{});
    else by_type(std::integral_constant<int, 256>{});
    return hipGetLastError();
}

}  // namespace cellm
