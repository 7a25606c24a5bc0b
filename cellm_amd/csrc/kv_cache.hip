// The 8-bit paged K/V cache: written from f32 K and V, read back, and, as the f16
// cache, compacted to the accepted path of a drafted tree (gfx950).
//
// A head vector x[HD] of one token is held as int8 codes and one f32 scale:
//   s = f32(max|x| / 127), c = clamp(rint(f32(x / s)), -127, 127), value = c * s
// so a value is off by at most s / 2 (and x by the rounding of the quotient, 2^-24 of it).
// s is 0 and so are the codes where max|x| / 127 is below the smallest normal f32: its
// quotients would be as coarse as the codes.  A vector with an infinity or a NaN gets the
// scale NaN and codes 0: it reads back as NaN, where f16 pages would show the element.
// Pages are head-major: vector (block, layer, kv head h, slot) is number
//   ((block * n_layers + layer) * n_kv + h) * tpb + slot
// of both arrays, so a head's positions of a page are one run of codes and one of scales
// and an attention block reads whole 128-byte lines, which the f16 cache's token-major
// order does not give heads of 64 codes.
//
// All three are bound by bytes or, where there are few, by their launch and the chain position -> page -> data.  Write: a
// team of lanes per head vector, 32 bytes of f32 a lane, the maximum by lane exchanges, so that a vector is read once;
// 2048 tokens of 32/8 heads of 128 with RoPE move 89 MB in 20 us, 4.5 TB/s (large copies: 4.7 to 5.3); one token of 9/3
// heads of 64 takes 3.4 us.
// Read: 16 bytes of output a thread; 8000 tokens of 8 heads of 128 to f16 move 50 MB in 10.3 us, 4.8 TB/s.  The move of
// accepted tokens: 4.1 us for 24 layers of 2 heads of 64, 4.6 for 32 layers of 8 heads of 128 in 8 sessions (5.4 MB).
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

#pragma clang fp contract(off)  // RoPE's products and sums are rounded one by one, as in decode.hip

namespace cellm {

namespace {

constexpr int kThreads = 256;

// vector number of token `slot` of row table `table` for head 0, or -1: no position, or its page is missing
__device__ __forceinline__ long long vector_of(const KvGeom& g, int table, int slot)
{
    if (slot < 0) return -1;
    const int b = slot / g.tpb;
    if (b >= g.max_blocks) return -1;
    const uint32_t blk = g.bt[(size_t)table * g.max_blocks + b];
    if (blk >= (uint32_t)g.total_blocks) return -1;
    return ((long long)blk * g.n_layers + g.layer) * g.n_kv * (long long)g.tpb + (slot - b * g.tpb);
}

struct WriteArgs {
    const float* q;       // nullptr: no q
    const float* k;
    const float* v;
    float* q_out;
    const float2* cs;     // nullptr: no rotation
    int table_positions, il;
    const int32_t* pos;
    const int32_t* slots;
    int rows, per, n_heads;
    int8_t* kc;
    float* ks;
    int8_t* vc;
    float* vs;
    KvGeom g;
};

// One team of HD / 8 lanes per head vector: a row's query heads, then its K heads, then its
// V heads.  Lane l holds 8 elements: the rotate-half pairs 4 l .. 4 l + 3, or (interleaved
// pairs, and V) elements 8 l .. 8 l + 7.
template <int HD>
__global__ __launch_bounds__(kThreads) void kv_write_q8_kernel(const WriteArgs a)
{
    constexpr int T = HD / 8, H = HD / 2;
    const int nq = a.q ? a.n_heads : 0, per_row = nq + 2 * a.g.n_kv;
    const int l = threadIdx.x % T;
    const uint32_t vec = blockIdx.x * (kThreads / T) + threadIdx.x / T;  // 32 bits: the host checks the count
    if (vec >= (uint32_t)a.rows * (uint32_t)per_row) return;  // whole teams
    const int r = (int)(vec / (uint32_t)per_row), h = (int)(vec - (uint32_t)r * (uint32_t)per_row);
    const bool is_q = h < nq, is_v = h >= nq + a.g.n_kv;
    const int kvh = is_q ? 0 : is_v ? h - nq - a.g.n_kv : h - nq;
    const int p = a.pos[r], slot = a.slots ? a.slots[r] : p;
    if (p < 0) return;
    const bool split = a.cs && !a.il && !is_v;  // rotate-half: two runs of four
    const int e0 = split ? 4 * l : 8 * l, e1 = split ? H + 4 * l : 8 * l + 4;
    const float* src = is_q ? a.q + ((size_t)r * a.n_heads + h) * HD
                            : (is_v ? a.v : a.k) + ((size_t)r * a.g.n_kv + kvh) * HD;
    const f4_t x0 = *reinterpret_cast<const f4_t*>(src + e0), x1 = *reinterpret_cast<const f4_t*>(src + e1);
    float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    if (a.cs && !is_v) {
        const int pp = min(p, a.table_positions - 1);
        const f4_t* cs = reinterpret_cast<const f4_t*>(a.cs + (size_t)pp * H + 4 * l);
        const f4_t c0 = cs[0], c1 = cs[1];
        const float co[4] = {c0[0], c0[2], c1[0], c1[2]}, si[4] = {c0[1], c0[3], c1[1], c1[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = split ? i : 2 * i, w = split ? 4 + i : 2 * i + 1;
            const float lo = x[u], hi = x[w];
            x[u] = lo * co[i] - hi * si[i];
            x[w] = hi * co[i] + lo * si[i];
        }
    }
    if (is_q) {
        float* dst = a.q_out + ((size_t)r * a.n_heads + h) * HD;
        *reinterpret_cast<f4_t*>(dst + e0) = f4_t{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f4_t*>(dst + e1) = f4_t{x[4], x[5], x[6], x[7]};
        return;
    }
    const long long v0 = vector_of(a.g, r / a.per, slot);
    if (v0 < 0) return;  // the same for the whole team
    uint32_t m = 0;      // |x| in the order of its bits: NaN above infinity above the finite
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
    m = team_max_u32<T>(m);
    float s = __builtin_bit_cast(float, m) / 127.0f;
    if (!(s >= 1.1754943508222875e-38f)) s = 0.0f;
    s = fminf(s, 0x1.0204060000000p+121f);  // 127 of it are finite: the quotient of the largest f32 is rounded up
    const bool finite = m < 0x7F800000u;
    uint32_t w[2] = {0, 0};
    if (finite && s > 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = (int)fminf(fmaxf(rintf(x[i] / s), -127.0f), 127.0f);
            w[i >> 2] |= (uint32_t)(c & 0xFF) << (8 * (i & 3));
        }
    }
    const size_t vn = (size_t)v0 + (size_t)kvh * a.g.tpb;
    int8_t* dst = (is_v ? a.vc : a.kc) + vn * HD;
    *reinterpret_cast<uint32_t*>(dst + e0) = w[0];
    *reinterpret_cast<uint32_t*>(dst + e1) = w[1];
    if (l == 0) (is_v ? a.vs : a.ks)[vn] = finite ? s : __builtin_nanf("");
}

__device__ __forceinline__ uint16_t bf16_rne(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0x7FC0;
    return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1u)) >> 16);
}

// E codes per thread, one 16-byte store of the output (eight 2-byte or four 4-byte values); a row
// whose position is missing reads as zeros, one without a position is left as it was.
template <int HD, int DT>
__global__ __launch_bounds__(kThreads) void kv_read_q8_kernel(const int8_t* __restrict__ kc, const float* __restrict__ ks,
                                                              const int8_t* __restrict__ vc, const float* __restrict__ vs,
                                                              const int32_t* __restrict__ pos, int rows, int per, KvGeom g,
                                                              void* __restrict__ ko, void* __restrict__ vo)
{
    constexpr int E = DT == DT_F32 ? 4 : 8, T = HD / E;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;  // 32 bits: the host checks the count
    if (i >= (uint32_t)rows * (uint32_t)g.n_kv * T) return;
    const uint32_t vec = i / T, row = vec / (uint32_t)g.n_kv;
    const int l = (int)(i % T), kvh = (int)(vec - row * (uint32_t)g.n_kv), r = (int)row;
    const int p = pos[r];
    if (p < 0) return;
    const long long v0 = vector_of(g, r / per, p);
    const size_t vn = v0 < 0 ? 0 : (size_t)v0 + (size_t)kvh * g.tpb;
    const auto one = [&](const int8_t* c, const float* s, void* out) {
        uint32_t w[E / 4];
        const uint32_t* src = reinterpret_cast<const uint32_t*>(c + vn * HD + E * l);
#pragma unroll
        for (int j = 0; j < E / 4; ++j) w[j] = src[j];
        const float sc = v0 < 0 ? 0.0f : s[vn];
        float x[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            x[j] = (float)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * sc;
            // the f32 value is what f16 rounds (a fused v_fma_mixlo_f16 would round the exact product); not volatile:
            // a volatile asm is a scheduling barrier
            if constexpr (DT == DT_F16) asm("" : "+v"(x[j]));
        }
        u4_t o;
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __builtin_bit_cast(uint32_t, x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint16_t a, b;
                if constexpr (DT == DT_F16) {
                    a = __builtin_bit_cast(uint16_t, (_Float16)x[2 * j]);
                    b = __builtin_bit_cast(uint16_t, (_Float16)x[2 * j + 1]);
                } else {
                    a = bf16_rne(x[2 * j]);
                    b = bf16_rne(x[2 * j + 1]);
                }
                o[j] = (uint32_t)a | (uint32_t)b << 16;
            }
        }
        reinterpret_cast<u4_t*>(out)[i] = o;
    };
    one(kc, ks, ko);
    one(vc, vs, vo);
}

// ---- the accepted path of a drafted tree ----------------------------------------------
// Slot ctx + i takes the K and V of slot ctx + accepted[i], in every layer.  The nodes of a
// path rise (a parent comes before its child), so accepted[i] >= i and no slot is written
// before it is read, by a thread that owns its column of every token and goes along the path.
struct AcceptArgs {
    unsigned char* a[2];   // K and V: rows of `row` bytes at ((block * units + unit) * tpb + slot) * row
    float* s[2];           // scales, one per row (8-bit pages), or null
    const int32_t* ctx;
    const int32_t* accepted;
    int most, tree, tpb, max_blocks, total_blocks, units, row;
    const uint32_t* bt;
};

constexpr int kPathStep = 8;  // tokens of a path in registers at a time

__global__ __launch_bounds__(kThreads) void kv_accept_kernel(const AcceptArgs a)
{
    __shared__ long long at[2][kMaxTree];  // row numbers of unit 0, source and target; -1: not moved
    __shared__ int count;
    const int t = threadIdx.x, table = blockIdx.y, ctx = a.ctx[table];
    const int32_t* path = a.accepted + (size_t)table * a.most;
    if (ctx < 0) return;  // the same for the whole block
    if (t == 0) count = a.most;
    __syncthreads();
    const auto row_of = [&](int node) {
        const long long p = (long long)ctx + node;
        const long long b = p / a.tpb;
        if (b >= a.max_blocks) return -1ll;
        const uint32_t blk = a.bt[(size_t)table * a.max_blocks + b];
        if (blk >= (uint32_t)a.total_blocks) return -1ll;
        return (long long)blk * a.units * a.tpb + (p - b * a.tpb);
    };
    for (int i = t; i < a.most; i += kThreads) {
        const int node = path[i], before = i ? path[i - 1] : -1;
        const bool ok = node >= 0 && node > before && node < a.tree;
        if (!ok) atomicMin(&count, i);  // the path ends at its first entry that is none
        const long long from = ok ? row_of(node) : -1, to = ok ? row_of(i) : -1;
        at[0][i] = from == to || to < 0 ? -1 : from;
        at[1][i] = to;
    }
    __syncthreads();
    const int n = count, cols = a.row / (int)sizeof(u4_t);
    const long long c = (long long)blockIdx.x * kThreads + t;
    const int unit = (int)(c / cols), col = (int)(c - (long long)unit * cols);
    if (unit >= a.units) return;
    for (int i0 = 0; i0 < n; i0 += kPathStep) {
        u4_t x[2][kPathStep];
        float sc[2][kPathStep];
#pragma unroll
        for (int j = 0; j < kPathStep; ++j) {
            const long long from = i0 + j < n ? at[0][i0 + j] : -1;
            const size_t row = from < 0 ? 0 : (size_t)from + (size_t)unit * a.tpb;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                x[w][j] = *reinterpret_cast<const u4_t*>(a.a[w] + row * a.row + (size_t)col * sizeof(u4_t));
                if (a.s[w] && col == 0) sc[w][j] = a.s[w][row];
            }
        }
#pragma unroll
        for (int j = 0; j < kPathStep; ++j) {
            if (i0 + j >= n || at[0][i0 + j] < 0) continue;
            const size_t row = (size_t)at[1][i0 + j] + (size_t)unit * a.tpb;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                *reinterpret_cast<u4_t*>(a.a[w] + row * a.row + (size_t)col * sizeof(u4_t)) = x[w][j];
                if (a.s[w] && col == 0) a.s[w][row] = sc[w][j];
            }
        }
    }
}

}  // namespace

hipError_t launch_kv_write_q8(const float* q, const float* k, const float* v, float* q_out, int rows, int per, int n_heads,
                              int head_dim, const int32_t* pos, const int32_t* slots, const float* cos_sin,
                              int table_positions, int interleaved, int8_t* kc, float* ks, int8_t* vc, float* vs,
                              const KvGeom& g, hipStream_t st)
{
    WriteArgs a{q, k, v, q_out, reinterpret_cast<const float2*>(cos_sin), table_positions, interleaved, pos, slots,
                rows, per, n_heads, kc, ks, vc, vs, g};
    const long long vecs = (long long)rows * ((q ? n_heads : 0) + 2 * g.n_kv);
    const auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value, V = kThreads / (HD / 8);
        hipLaunchKernelGGL((kv_write_q8_kernel<HD>), dim3((unsigned)((vecs + V - 1) / V)), dim3(kThreads), 0, st, a);
    };
    if (head_dim == 64) go(std::integral_constant<int, 64>{});
    else if (head_dim == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return hipGetLastError();
}

hipError_t launch_kv_read_q8(const int8_t* kc, const float* ks, const int8_t* vc, const float* vs, const int32_t* pos,
                             int rows, int per, int head_dim, const KvGeom& g, void* k_out, void* v_out, int out_dtype,
                             hipStream_t st)
{
    const auto go = [&](auto hd, auto dt) {
        constexpr int HD = decltype(hd)::value, DT = decltype(dt)::value, T = HD / (DT == DT_F32 ? 4 : 8);
        const long long n = (long long)rows * g.n_kv * T;
        hipLaunchKernelGGL((kv_read_q8_kernel<HD, DT>), dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                           st, kc, ks, vc, vs, pos, rows, per, g, k_out, v_out);
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

hipError_t launch_kv_accept(void* kc, float* ks, void* vc, float* vs, int units, int row_bytes, int tables,
                            const int32_t* ctx, const int32_t* accepted, int most, int tree, int tpb, int max_blocks,
                            int total_blocks, const uint32_t* bt, hipStream_t st)
{
    AcceptArgs a{{static_cast<unsigned char*>(kc), static_cast<unsigned char*>(vc)}, {ks, vs}, ctx, accepted, most, tree,
                 tpb, max_blocks, total_blocks, units, row_bytes, bt};
    const long long n = (long long)units * (row_bytes / (int)sizeof(u4_t));  // rows are whole words: head_dim is 64 or more
    hipLaunchKernelGGL(kv_accept_kernel, dim3((unsigned)((n + kThreads - 1) / kThreads), (unsigned)tables), dim3(kThreads), 0,
                       st, a);
    return hipGetLastError();
}

}  // namespace cellm
