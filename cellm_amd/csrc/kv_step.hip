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
//
// Latency bounds it: one block goes over the sessions, a thread each, and what differs in size from session to
// session (a finished one's pages, a prompt's) is shared out flat, an entry a thread, by a search in the running
// sums (four entries a thread: 11.3 us for 11.8 where 13 sessions give 1600 pages back, but 6.9 for 5.8 where few do).
// The rows' positions and slots are filled by the same block where they are few, else by a second launch over
// the whole chip (kFillRows).  8 sessions that take a token each 4.4 us, 256 with 24 prompts 11.8, 64 prompts of 64 thousand
// rows 8.4 (one thread per session for all of its pages, and one block for all rows: 6.6, 22 and 73).
constexpr int kFillRows = 2048;      // 256 sessions: 1024 rows 6.7 us in one launch and 8.2 in two, 4096 9.4 and 8.4, 8192 20.1 and 11.9
constexpr int kPlanSmall = 256;      // sessions for which a block of 256 threads is launched, not of 1024: 5.8 us at 256, 8.0
constexpr int kFillThreads = 256;
constexpr int kFillSessions = 4096;  // of which the filling blocks hold the row starts in LDS

// Running sum of v over the block's threads; sums: a word per wave.  All threads get the block's total.
template <int N, typename T>
__device__ __forceinline__ T block_scan(T v, T* sums, T& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = 1; o < 64; o <<= 1) {
        const T u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < N / 64; ++w) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    return v + before;
}

// The first of n rising sums that is above i
__device__ __forceinline__ int above(const uint32_t* sums, int n, uint32_t i)
{
    int lo = 0;
    for (int step = n >> 1; step; step >>= 1)  // n: a power of two
        if (sums[lo + step - 1] <= i) lo += step;
    return lo;
}

__device__ __forceinline__ int slot_of(const KvPlanArgs& a, int session, int pos)
{
    const int b = pos / a.tpb;
    const uint32_t blk = a.bt[(size_t)session * a.max_blocks + b];
    return blk < (uint32_t)a.total_blocks ? (int)(blk * (uint32_t)a.tpb) + (pos - b * a.tpb) : -1;
}

// N threads; FILL: the rows too
template <int N, bool FILL>
__global__ __launch_bounds__(N) void kv_plan_kernel(const KvPlanArgs a)
{
    __shared__ uint32_t sums[N], row_sums[FILL ? N : 1], wave_sums[N / 64];
    __shared__ unsigned long long wave_pairs[N / 64];
    __shared__ int held_of[N], lens_of[FILL ? N : 1];
    __shared__ uint32_t last[2];   // pages and rows of the last session that fits
    const int t = threadIdx.x, lane = t & 63;
    const auto pages_of = [&](long long tokens) { return (uint32_t)((tokens + a.tpb - 1) / a.tpb); };
    long long count = max(a.free_count[0], 0);
    if (count > a.free_capacity) count = a.free_capacity;
    int ctx = t < a.tables ? a.ctx[t] : -1, add = t < a.tables ? a.add[t] : 0;  // of the round at hand

    // ---- finished sessions give their pages back, in the order of sessions and positions
    for (int t0 = 0; t0 < a.tables; t0 += N) {
        if (t0) {
            const int s = t0 + t;
            ctx = s < a.tables ? a.ctx[s] : -1;
            add = s < a.tables ? a.add[s] : 0;
        }
        const uint32_t entries = ctx >= 0 && add < 0 ? min(pages_of(ctx), (uint32_t)a.max_blocks) : 0;
        if (!__syncthreads_or(entries > 0)) continue;
        uint32_t all;
        sums[t] = block_scan<N>(entries, wave_sums, all);
        for (uint32_t i0 = 0; i0 < all; i0 += N) {
            __syncthreads();
            const uint32_t i = i0 + t;
            uint32_t blk = ~0u, n;
            if (i < all) {
                const int s = above(sums, N, i);
                blk = a.bt[(size_t)(t0 + s) * a.max_blocks + (i - (s ? sums[s - 1] : 0))];
            }
            const uint32_t there = blk < (uint32_t)a.total_blocks ? 1 : 0;
            const long long at = count + block_scan<N>(there, wave_sums, n) - 1;
            if (there && at < a.free_capacity) a.free_blocks[at] = blk;
            count = min(count + n, (long long)a.free_capacity);
        }
    }
    __syncthreads();  // the free list as it is now
    if (a.tables > N) {
        ctx = a.ctx[t];
        add = a.add[t];
    }

    // ---- sessions in order, up to the first whose pages or rows are not there
    long long pages0 = 0, rows0 = 0;  // of the sessions before this round's
    if (t == 0) a.starts[0] = 0;
    for (int t0 = 0; t0 < a.tables; t0 += N) {
        const int s = t0 + t;
        if (t0) {
            ctx = s < a.tables ? a.ctx[s] : -1;
            add = s < a.tables ? a.add[s] : 0;
        }
        const bool valid = ctx >= 0 && add > 0 && (long long)ctx + add <= (long long)a.max_blocks * a.tpb;
        const uint32_t held = ctx > 0 ? pages_of(ctx) : 0;
        const uint32_t need = valid ? pages_of((long long)ctx + add) - held : 0;
        const uint32_t asked = valid ? (uint32_t)min(add, a.rows + 1) : 0;
        // both sums stay below 2^31: 2^20 pages or rows and one of each of 1024 sessions
        unsigned long long all;
        const unsigned long long up = block_scan<N>((unsigned long long)need << 32 | asked, wave_pairs, all);
        const uint32_t p = (uint32_t)(up >> 32), r = (uint32_t)up;
        const bool fits = pages0 + p <= count && rows0 + r <= a.rows;
        if (t < 2) last[t] = 0;
        __syncthreads();
        const unsigned long long in = __ballot(fits);
        if (in && lane == 63 - __builtin_clzll(in)) {  // sums rise with the sessions
            atomicMax(&last[0], p);
            atomicMax(&last[1], r);
        }
        __syncthreads();
        const uint32_t pages = last[0], rows = last[1];
        const int len = fits && valid ? ctx + add : ctx >= 0 && add < 0 ? 0 : ctx;
        sums[t] = fits ? p : pages;
        held_of[t] = (int)(held + (fits ? need : 0) - sums[t]);  // entry of page i: held_of + i, of a session that has it
        if constexpr (FILL) {
            row_sums[t] = fits ? r : rows;
            lens_of[t] = len - (int)row_sums[t];
        }
        if (s < a.tables) {
            a.starts[s + 1] = (int32_t)(rows0 + (fits ? r : rows));
            a.lens_out[s] = len;
        }
        __syncthreads();
        for (uint32_t i = t; i < pages; i += N) {
            const int e = above(sums, N, i);
            a.bt[(size_t)(t0 + e) * a.max_blocks + (held_of[e] + (int)i)] = a.free_blocks[count - 1 - (pages0 + i)];
        }
        __syncthreads();
        if constexpr (FILL) {
            for (uint32_t i = t; i < rows; i += N) {
                const int e = above(row_sums, N, i), pos = lens_of[e] + (int)i;
                a.pos[rows0 + i] = pos;
                a.slots[rows0 + i] = slot_of(a, t0 + e, pos);
            }
        }
        pages0 += pages;
        rows0 += rows;
        if (!__syncthreads_and(fits)) {  // nothing more fits: the others wait
            for (int e = t0 + N + t; e < a.tables; e += N) {
                const int c = a.ctx[e];
                a.starts[e + 1] = (int32_t)rows0;
                a.lens_out[e] = c >= 0 && a.add[e] < 0 ? 0 : c;
            }
            break;
        }
    }
    if (t == 0) a.free_out[0] = (int32_t)(count - pages0);
    if constexpr (FILL) {
        for (long long i = rows0 + t; i < a.rows; i += N) {
            a.pos[i] = -1;
            a.slots[i] = -1;
        }
    }
}

// Positions and slots of many rows, a row a thread, once the sessions have theirs.
__global__ __launch_bounds__(kFillThreads) void kv_fill_kernel(const KvPlanArgs a)
{
    __shared__ int32_t lds[kFillSessions + 1];
    const bool small = a.tables <= kFillSessions;
    if (small) {
        for (int i = threadIdx.x; i <= a.tables; i += kFillThreads) lds[i] = a.starts[i];
        __syncthreads();
    }
    const auto start = [&](int t) { return small ? lds[t] : a.starts[t]; };
    const int r = (int)(blockIdx.x * kFillThreads + threadIdx.x);
    if (r >= a.rows) return;
    int pos = -1, slot = -1;
    if (r < start(a.tables)) {
        int lo = 0, hi = a.tables;  // start(lo) <= r < start(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start(mid) <= r) lo = mid;
            else hi = mid;
        }
        pos = a.lens_out[lo] - (start(lo + 1) - r);
        slot = slot_of(a, lo, pos);
    }
    a.pos[r] = pos;
    a.slots[r] = slot;
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
    const auto go = [&](auto n, auto fill) {
        constexpr int N = decltype(n)::value;
        hipLaunchKernelGGL((kv_plan_kernel<N, decltype(fill)::value>), dim3(1), dim3(N), 0, st, a);
    };
    const auto by_size = [&](auto fill) {
        if (a.tables <= kPlanSmall) go(std::integral_constant<int, 256>{}, fill);
        else go(std::integral_constant<int, 1024>{}, fill);
    };
    if (a.rows <= kFillRows) {
        by_size(std::true_type{});
    } else {
        by_size(std::false_type{});
        hipLaunchKernelGGL(kv_fill_kernel, dim3((unsigned)((a.rows + kFillThreads - 1) / kFillThreads)), dim3(kFillThreads), 0, st, a);
    }
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
