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

// n / d by the upper half of a product with 2^(32 + shift) / d rounded up: n below 2^31
struct Divisor {
    uint32_t mul;
    int shift;  // -1: d is 1
};
Divisor divisor_of(uint32_t d)
{
    int shift = -1;
    while (1ull << (shift + 1) < d) ++shift;
    return {shift < 0 ? 0u : (uint32_t)(((1ull << (32 + shift)) + d - 1) / d), shift};
}
__device__ __forceinline__ uint32_t over(uint32_t n, Divisor d)
{
    return d.shift < 0 ? n : __umulhi(n, d.mul) >> d.shift;
}

// ---- the pages and rows of a step -----------------------------------------------------
// Session t holds ctx tokens in ceil(ctx / tpb) pages and asks for `add` more.  With running sums
// over the sessions, P of the pages that these need and R of their rows,
//   it gets them where P <= pages free and R <= rows: in order, up to the first that does not fit.
// Page i of those handed out (counted over the sessions) is entry count - 1 - i of the free
// list, after the pages of finished sessions (add < 0) have been put onto its end.
//
// Latency bounds it: one block goes over the sessions, a thread each, and what differs in size from session to
// session (a finished one's pages, a prompt's) is shared out flat, an entry a thread, by a search in the running
// sums (four entries a thread of 256: 11.3 us for 11.8 where 13 sessions give 1600 pages back, but 6.9 for 5.8 where few do).
// The rows' positions and slots are filled by the same block where they are few, else by a second launch over
// the whole chip (kFillRows).  8 sessions that take a token each 4.4 us, 256 with 24 prompts 10.6, 64 prompts of 64 thousand
// rows 7.8 (one thread per session for all of its pages, and one block for all rows: 6.6, 22 and 73).
constexpr int kFillRows = 2048;      // 256 sessions: 1024 rows 6.7 us in one launch and 8.2 in two, 4096 9.4 and 8.9, 8192 20.1 and 10.6
constexpr int kPlanSmall = 256;      // sessions for which a block has so many threads, not 1024: 5.7 us at 256, 8.0 (512 threads: 6.2)
constexpr int kPlanMany = 512;       // and where rows are many, with as many pages: 256 sessions with 24 prompts 10.6, 256 threads 11.8, 1024 11.5
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
    int ctx = t < a.tables ? a.ctx[t] : -1, add = t < a.tables ? a.add[t] : 0;  // of the turn at hand

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
    long long pages0 = 0, rows0 = 0;  // of the sessions of earlier turns
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
template <int O>
__device__ __forceinline__ double lane_xor64(double v)
{
    const u2_t b = __builtin_bit_cast(u2_t, v);
    const auto half = [](uint32_t w) { return __builtin_bit_cast(uint32_t, lane_xor<O>(__builtin_bit_cast(float, w), 64)); };
    return __builtin_bit_cast(double, u2_t{half(b[0]), half(b[1])});
}
template <int T>
__device__ __forceinline__ double team_sum64(double v)
{
    if constexpr (T >= 32) v += lane_xor64<16>(v);
    if constexpr (T >= 16) v += lane_xor64<8>(v);
    v += lane_xor64<4>(v);
    v += lane_xor64<2>(v);
    return v + lane_xor64<1>(v);
}
// 1 / sqrt(m) to some 2^-50: the approximate one y (2^-24 and better) and the first two terms of (1 - e)^(-1/2),
// e = 1 - m y^2.
__device__ __forceinline__ double inv_sqrt64(double m)
{
    const double y = __builtin_amdgcn_rsq(m);
    const double e = __builtin_fma(-(m * y), y, 1.0);
    const double z = __builtin_fma(y * e, __builtin_fma(0.375, e, 0.5), y);
    return m > 0.0 && m < __builtin_inf() ? z : y;
}
// Four weights as they lie in memory, and as floats
template <int WDT>
using Raw4 = std::conditional_t<WDT == DT_F32, u4_t, u2_t>;
template <int WDT>
__device__ __forceinline__ f4_t floats(Raw4<WDT> w)
{
    if constexpr (WDT == DT_F32) {
        return __builtin_bit_cast(f4_t, w);
    } else if constexpr (WDT == DT_F16) {
        const h2_t a = as_h2(w[0]), b = as_h2(w[1]);
        return f4_t{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
    } else {
        const auto f = [](uint32_t u) { return __builtin_bit_cast(float, u); };
        return f4_t{f(w[0] << 16), f(w[0] & 0xFFFF0000u), f(w[1] << 16), f(w[1] & 0xFFFF0000u)};
    }
}

struct NormWriteArgs {
    NormRopeArgs n;
    int rows, n_heads;
    Divisor per_row, tokens;  // heads of a row, tokens of a page
    int tpb, layer, n_layers, n_kv;
    uint32_t slots_end;
};

// One team of HD / 8 lanes per head vector: a row's query heads, then its K heads, then its V heads.  Lane l holds dims
// 4 l .. 4 l + 3 and HD / 2 + 4 l .. HD / 2 + 4 l + 3: the pairs of the rotate-half layout, two pairs of each run of
// the interleaved one, and 8 lanes hold two groups of 4-bit codes.
//
// Bytes bound it at many rows, latency at few.  Back to back, 2048 rows of 32/8/8 heads of 128 to 8-bit pages (89 MB)
// take 18.4 us, 4.9 TB/s where a copy of 256 MiB reaches 5.4 (15.9 called one by one, when half of the reads come out of
// the cache); to 4-bit pages 17.4, to f16 ones 19.7; 7996 rows of 4/1/1 heads of 256 to 4-bit pages (93 MB) 18.3, to f16
// ones 17.7; one row 2.4.  A vector's loads are all on their way before its position and slot are looked at, the sum goes round by lane
// moves, quotients by integers are products, codes take no division, and of 4-bit codes two lanes share out their two
// words (shuffles, divisions and 2-byte stores took 9 % more, 13 % of 4-bit pages and of one row); rows in order within each XCD read the table
// of cosines from its own L2 (7996 rows written and read back 25.5 us, 26.1 with blocks dealt out in turn).
template <int HD, int FMT, int WDT>
__global__ __launch_bounds__(kThreads) void norm_rope_write_kernel(const NormWriteArgs A)
{
    constexpr int T = HD / 8, H = HD / 2;
    const NormRopeArgs& a = A.n;
    const int per_row = A.n_heads + 2 * A.n_kv, l = threadIdx.x % T;
    const uint32_t block = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);  // each XCD has rows that follow one another
    const uint32_t vec = block * (kThreads / T) + threadIdx.x / T;  // the host checks the count
    if (vec >= (uint32_t)A.rows * (uint32_t)per_row) return;              // whole teams
    const int r = (int)over(vec, A.per_row), h = (int)(vec - (uint32_t)r * (uint32_t)per_row);
    const bool is_q = h < A.n_heads, is_v = h >= A.n_heads + A.n_kv;
    const int kvh = is_q ? 0 : is_v ? h - A.n_heads - A.n_kv : h - A.n_heads;
    const int p = a.pos[r];
    const uint32_t slot = (uint32_t)a.slots[r];
    const int e0 = 4 * l, e1 = H + 4 * l;
    const float* src = is_q ? a.q + ((size_t)r * A.n_heads + h) * HD
                            : (is_v ? a.v : a.k) + ((size_t)r * A.n_kv + kvh) * HD;
    const f4_t x0 = *reinterpret_cast<const f4_t*>(src + e0), x1 = *reinterpret_cast<const f4_t*>(src + e1);
    const void* weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    Raw4<WDT> w0 = {}, w1 = {};
    if (weight) {
        w0 = static_cast<const Raw4<WDT>*>(weight)[e0 / 4];
        w1 = static_cast<const Raw4<WDT>*>(weight)[e1 / 4];
    }
    if (p < 0 || (!is_q && slot >= A.slots_end)) return;
    const bool turned = a.cos_sin && !is_v;
    f4_t c0 = {}, c1 = {};  // (cos, sin) of two pairs each
    if (turned) {
        const float* cs = a.cos_sin + (size_t)min(p, a.table_positions - 1) * HD;
        c0 = *reinterpret_cast<const f4_t*>(cs + (a.interleaved ? e0 : 8 * l));
        c1 = *reinterpret_cast<const f4_t*>(cs + (a.interleaved ? e1 : 8 * l + 4));
    }
    float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    if (weight) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)x[i], (double)x[i], ss);
        const f4_t y0 = floats<WDT>(w0), y1 = floats<WDT>(w1);
        const float inv = (float)inv_sqrt64(team_sum64<T>(ss) * (1.0 / HD) + (double)a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = x[i] * inv;
            x[i] = y * (i < 4 ? y0[i] : y1[i - 4]);
        }
    }
    if (turned) {
        const auto turn = [&](int u, int w, float co, float si) {
            const float lo = x[u], hi = x[w];
            x[u] = lo * co - hi * si;
            x[w] = hi * co + lo * si;
        };
        if (!a.interleaved) {
            turn(0, 4, c0[0], c0[1]);
            turn(1, 5, c0[2], c0[3]);
            turn(2, 6, c1[0], c1[1]);
            turn(3, 7, c1[2], c1[3]);
        } else {
            turn(0, 1, c0[0], c0[1]);
            turn(2, 3, c0[2], c0[3]);
            turn(4, 5, c1[0], c1[1]);
            turn(6, 7, c1[2], c1[3]);
        }
    }
    if (is_q) {
        float* dst = a.q_out + ((size_t)r * A.n_heads + h) * HD;
        *reinterpret_cast<f4_t*>(dst + e0) = f4_t{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f4_t*>(dst + e1) = f4_t{x[4], x[5], x[6], x[7]};
        return;
    }
    const uint32_t blk = over(slot, A.tokens), off = slot - blk * (uint32_t)A.tpb;
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
        uint32_t* dst = static_cast<uint32_t*>(is_v ? a.vc : a.kc) + vn * (HD / 8);
        uint32_t* sc = static_cast<uint32_t*>(is_v ? a.vs : a.ks) + vn * (HD / 32);
        uint32_t w[2], s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float y[4] = {x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]};
            w[u] = quantise4(y, s[u]);
        }
        // of two lanes the even one stores their word of the first half, the odd one that of the second
        const bool odd = l & 1;
        const uint32_t other = __builtin_bit_cast(uint32_t, dpp_xor1(__builtin_bit_cast(float, odd ? w[0] : w[1])));
        dst[(odd ? H / 8 : 0) + l / 2] = odd ? other | w[1] << 16 : w[0] | other << 16;
        if (l % 8 < 2) sc[(odd ? H / 32 : 0) + l / 8] = odd ? s[1] : s[0];
    }
}

// ---- 4-bit pages read back --------------------------------------------------------------
struct ReadArgs {
    const void *kc, *ks, *vc, *vs;
    const int32_t* pos;
    void *ko, *vo;
    KvGeom g;
    int rows;
    Divisor heads, per, tokens;  // of a row, rows of a table, of a page
};

// E codes of K and of V per thread, one 16-byte store of each.  The outputs' bytes bound it, and at the sizes of a step the
// way there, position, page, codes: 7996 rows of one head of 256 to f32 (19 MB) 5.9 us, 7.3 with a word of codes and
// 32 bytes out per thread.
template <int HD, int DT>
__global__ __launch_bounds__(kThreads) void kv_read_q4_kernel(const ReadArgs A)
{
    constexpr int E = DT == DT_F32 ? 4 : 8, T = HD / E;
    const KvGeom& g = A.g;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;  // the host checks the count
    if (i >= (uint32_t)A.rows * (uint32_t)g.n_kv * T) return;
    const uint32_t vec = i / T, row = over(vec, A.heads), l = i % T, kvh = vec - row * (uint32_t)g.n_kv;
    const int p = A.pos[row];
    if (p < 0) return;
    const uint32_t b = over((uint32_t)p, A.tokens);
    uint32_t blk = ~0u;
    if (b < (uint32_t)g.max_blocks) blk = g.bt[(size_t)over(row, A.per) * g.max_blocks + b];
    const bool there = blk < (uint32_t)g.total_blocks;
    const size_t vn = (((size_t)blk * g.n_layers + g.layer) * g.n_kv + kvh) * g.tpb + ((uint32_t)p - b * (uint32_t)g.tpb);
    const auto one = [&](const void* codes, const void* scales, void* out) {
        uint32_t w = 0, m = 0;
        if (there) {
            if constexpr (E == 4) w = static_cast<const uint16_t*>(codes)[vn * T + l];
            else w = static_cast<const uint32_t*>(codes)[vn * T + l];
            m = static_cast<const uint32_t*>(scales)[vn * (HD / 32) + E * l / 32];
        }
        const h2_t s = as_h2(both_low(m)), z = as_h2(both_high(m));
        u4_t o;
        if constexpr (E == 4) {
            w |= w << 12;  // nibbles 0 and 1, 2 and 3 at bits 0 and 16, 8 and 24
            const h2_t a = values4(w & 0x000F000Fu, s, z), c = values4(w >> 8 & 0x000F000Fu, s, z);
            o = __builtin_bit_cast(u4_t, f4_t{(float)a[0], (float)a[1], (float)c[0], (float)c[1]});
        } else {
            _Float16 x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // nibbles j and j + 4
                const h2_t v = values4(w >> (4 * j) & 0x000F000Fu, s, z);
                x[j] = v[0];
                x[j + 4] = v[1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == DT_F16) o[j] = as_u32(h2_t{x[2 * j], x[2 * j + 1]});
                else o[j] = (uint32_t)bf16_rne((float)x[2 * j]) | (uint32_t)bf16_rne((float)x[2 * j + 1]) << 16;
            }
        }
        static_cast<u4_t*>(out)[i] = o;
    };
    one(A.kc, A.ks, A.ko);
    one(A.vc, A.vs, A.vo);
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t st)
{
    const auto go = [&](auto n, auto fill) {
        constexpr int N = decltype(n)::value;
        hipLaunchKernelGGL((kv_plan_kernel<N, decltype(fill)::value>), dim3(1), dim3(N), 0, st, a);
    };
    const auto by_size = [&](auto few, auto fill) {
        if (a.tables <= decltype(few)::value) go(few, fill);
        else go(std::integral_constant<int, 1024>{}, fill);
    };
    if (a.rows <= kFillRows) {
        by_size(std::integral_constant<int, kPlanSmall>{}, std::true_type{});
    } else {
        by_size(std::integral_constant<int, kPlanMany>{}, std::false_type{});
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
    a.slots_end = (uint32_t)std::min((long long)g.total_blocks * g.tpb, 1ll << 31);  // slots: numbers of 31 bits
    a.per_row = divisor_of((uint32_t)(n_heads + 2 * g.n_kv));
    a.tokens = divisor_of((uint32_t)g.tpb);
    const long long vecs = (long long)rows * (n_heads + 2 * g.n_kv);
    const auto go = [&](auto hd, auto fm, auto wt) {
        constexpr int HD = decltype(hd)::value, V = kThreads / (HD / 8);
        hipLaunchKernelGGL((norm_rope_write_kernel<HD, decltype(fm)::value, decltype(wt)::value>),
                           dim3((unsigned)((vecs + 8 * V - 1) / (8 * V) * 8)), dim3(kThreads), 0, st, a);
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
    const ReadArgs a{kc, ks, vc, vs, pos, k_out, v_out, g, rows, divisor_of((uint32_t)g.n_kv), divisor_of((uint32_t)per),
                     divisor_of((uint32_t)g.tpb)};
    const auto go = [&](auto hd, auto dt) {
        constexpr int HD = decltype(hd)::value, DT = decltype(dt)::value;
        const long long n = (long long)rows * g.n_kv * (HD / (DT == DT_F32 ? 4 : 8));
        hipLaunchKernelGGL((kv_read_q4_kernel<HD, DT>), dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                           st, a);
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
