// Attention over paged K/V whose pages many query rows share (gfx950): 8-bit pages for
// decode and prompts, and 8-bit or f16 pages for trees of drafted tokens.
//
//   s_p = scale * (q . k_p), capped: s = cap * tanh(s / cap)
//   o   = sum_p e^(s_p - M) v_p / sum_p e^(s_p - M),   M = max_p s_p
// over the positions p that the row sees: up to its own, the last `window` of them; or
// (trees) the context and, behind it, the drafted slots whose bit its mask has.  A missing
// page counts as zero keys and values.  8-bit keys and values are c * s with one scale per
// (token, kv head), which leaves both sums: q . k = s_k (q . c_k), and s_v joins the weight.
//
// The (row, query head) pairs of a table that read one kv head are its columns; a block
// computes 16 of them over a range of positions, so each K and V element is fetched once for
// all.  Its four waves take chunks of CH positions in turn and meet in LDS at the end:
//   S^T [CH][16 columns] = K . Q^T       O^T [HD][16 columns] += V^T . P^T
// Row m of a K tile is position 4 (m % 4) + m / 4 of its 16, which leaves lane (column c,
// group g) of S^T with positions 4 j + g, j = 0, 1, ...: the k order of the second product is
// free as long as V^T and P^T agree, so those weights are its B operand as they are, and the
// four groups of a V load read four neighbouring positions.  V^T needs a lane's row to be a
// dim: row c of tile e is dim c * HD / 16 + e, so lane c reads HD / 16 neighbouring dims of
// its positions and no V goes through LDS.
//
// 8-bit pages: q is held as integers of 2^-22 of its head's largest |q| (rounded to the
// nearest), as three signed 8-bit digits, and q . c_k is three exact sums on
// v_mfma_i32_16x16x64_i8 with the codes as they are.  A head whose largest element stands far
// above the others has a fourth digit, 2^-30 of the largest (kLoud).  f16 pages: q as two f16 parts, hi =
// RNE_f16(q') and lo = RNE_f16(q' - hi) of q scaled by a power of two (23 bits of an element,
// 2^-38 of the largest).  Scores, exponentials and sums are f32.
//
// Weights are powers of two, w = 2^(c s - R) (c s rounded by itself, so that scores too large for
// the difference to have bits still compare) with c = log2(e) times what of the score's scale
// is left out of s, against a reference R of each column that stands in for the maximum: l and
// O hold sums of w and of w s_v v, so any R gives the same quotient.  The products w s_v are
// two f16 parts like q's, over the codes as exact f16 integers or f16 values, and R is raised
// (and l and O with it) only where one of them passes 2^15, to leave the largest at 2^13: a
// test of the lanes' own values, where a maximum of each chunk would be sums over lanes.
//
// The positions of a set of columns are split over blocks by a rule on the device (plan()),
// which knows how long every context is; the last block of a set to finish adds the others'
// sums in split order.
//
// What bounds it (gfx950).  Decode: the reads and how they are shared out.  One session at 131072 positions, 32/8 heads of
// 128, takes 58 to 61 us for 277 MB, 4.7 TB/s; 8 sessions of 4096 to 8192 28 to 29 for 104 MB, 3.7 TB/s, with a block on
// 208 of the 256 CUs and walks of up to 9 units where 7 would do (a bare read of them takes 42 and 16.5; vector ALU
// busy 23 %, matrix units 6).  Short contexts: latency.  A block of one unit of positions takes 6.2 us (100 positions, 14/2
// heads of 64), each further one 1.8 (page entry, K, scores, weights, V one after the other): 9.7 at 701, unsplit.
// Many columns: vector instructions at two waves per SIMD (1024 tokens onto as many, 32/8 heads of 128, 84 us: vector ALU
// busy 62 %, matrix units 20 %, 307 TFLOP/s of the formula's products).
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"

#pragma clang fp contract(off)

namespace cellm {

namespace {

constexpr int kWaves = 4, kThreads = kWaves * 64, kCols = 16;
constexpr int kMaxSplits = 64;    // of a set's positions
// Sets of so many units of positions (a chunk for each wave) are not split: the meeting of splits costs about 4.5 us, a
// walk of three units less.  Units of 256 positions: 300 (14/2 heads of 64) 8.3 us, 10.8 in splits; 701 9.7 and 10.9; a
// tree of 16 nodes at 500 10.0 and 12.3; a prompt of 512 10.4 and 15.9.  At four units splits win: 1000 positions 10.9,
// 11.4 whole; 4 sessions of 1000, 32/8 heads of 128, 12.7 and 14.1.  Units of 128 (8-bit heads of 256, f16 of 128 and 256)
// walk faster: three units 12.5 us, 14.7 in splits (370 positions, 8/1 heads of 256), and four still lose in splits, 15.1
// to 14.1, and a tree of 16 nodes at 490 over f16 heads of 128 14.9 to 11.4.
constexpr int kWholeUnits = 3;
constexpr int kPlanSets = 256;    // sets that plan() looks at, 4 a lane: fewer than kPlanBlocks
// Splits aim at one block on each of the 256 CUs, though two run at once: fewer, longer walks keep the reads going and meet
// faster (one session at 131072 positions, 32/8 heads of 128: 61.3 us, 66.1 with 512 blocks; 16 sessions at 8000, 8/1
// heads of 256, 24.5 and 29.5; 300 rows at 600 of those 19.9 and 26.3).  Fewer stand than that: the sets are taken off
// for their last splits, which may be short, and the share is rounded up (8 sessions of 4096 to 8192 positions, 32/8
// heads of 128, 208 blocks; 24 such 192; 8 at 1000 positions 128, which have 15.3 us, and 13.8 under a bound of 512).
constexpr int kPlanBlocks = 256;
static_assert(kPlanSets >= kPlanBlocks);
// Sets of 32 columns where they leave at least so many blocks: each K and V tile serves twice the columns (8 trees of
// 63 nodes at 4096 positions, 32/8 heads of 128, f16: 90 us, 140 with 16 columns; a prompt of 1024 over 8-bit pages 90
// and 104), but with fewer blocks the chip stands idle (16 trees of 8 nodes at 1000 positions 32.1 us, 18.3 with 16
// columns; a prompt of 512 with 14/2 heads of 64 21.2 and 10.5; one f16 tree of 26 nodes 17.4 and 12.4).
constexpr int kWideBlocks = 256;

struct MmaArgs {
    PagedAttnArgs a;
    int group, cols, tiles, sets;  // heads per kv head; columns of a set; sets of a table, and of all tables
    int cap, tpb_shift;      // positions of a table; log2(tpb), or -1
    int want;                // blocks per kv head that plan() aims at; 0: one block per set
    uint32_t* counters;      // [set][kv head]: splits done, zero between calls
    float* part;             // [work][kv head]: [cols][HD] sums, [cols] references, [cols] sums of weights
    uint32_t part_bytes;
};

__device__ __forceinline__ bool finite_f32(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u; }
// Agent-coherent (sc1) stores and loads of a split's sums, 16 bytes at a time; offsets in floats.
constexpr int kSc1 = 16;
__device__ __forceinline__ void st_agent4(__amdgpu_buffer_rsrc_t r, uint32_t off, f4_t v)
{
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v), r, (int)(4u * off), 0, kSc1);
}
__device__ __forceinline__ f4_t ld_agent4(__amdgpu_buffer_rsrc_t r, uint32_t off)
{
    return __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(4u * off), 0, kSc1));
}
__device__ __forceinline__ void st_agent(__amdgpu_buffer_rsrc_t r, uint32_t off, float v)
{
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, (int)(4u * off), 0, kSc1);
}
__device__ __forceinline__ float ld_agent(__amdgpu_buffer_rsrc_t r, uint32_t off)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)(4u * off), 0, kSc1));
}
// LDS of one wave, written and read across its lanes: the wave's LDS operations run in order, and the
// compiler moves none across this
__device__ __forceinline__ void wave_lds_fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ int rfl(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What a row sees: positions start..ctx - 1, then (masks) those of ctx..end - 1 whose bit is set.
struct Sight {
    int start, ctx, end;
    const uint64_t* bits;
    __device__ __forceinline__ bool sees(int p) const
    {
        return p >= start && (p < ctx || (p < end && (bits[(p - ctx) >> 6] >> ((p - ctx) & 63) & 1)));
    }
};

__device__ __forceinline__ uint64_t tree_word(const PagedAttnArgs& a, const uint64_t* bits, int w)
{
    const int left = a.per - 64 * w;
    return bits[w] & (left >= 64 ? ~0ull : (1ull << left) - 1);
}

// false: the row has no position, or its mask no node, and its output is left as it was
__device__ __forceinline__ bool sight_of(const PagedAttnArgs& a, int cap, int table, int row, Sight& s)
{
    if (!a.masks) {
        const int p = a.pos[row];
        s.end = s.ctx = min(p, cap - 1) + 1;
        s.start = a.window > 0 ? max(s.ctx - a.window, 0) : 0;
        s.bits = nullptr;
        return p >= 0;
    }
    const int c = a.pos[table];
    int nodes = 0;
    s.bits = a.masks + (size_t)row * a.words;
    for (int w = 0; w < a.words; ++w) nodes += __popcll(tree_word(a, s.bits, w));
    s.ctx = min(c, cap);
    s.end = min(s.ctx + a.per, cap);
    // the node stands at position c + nodes - 1 (its ancestors and itself), in the table or past it; window >= nodes
    s.start = a.window > 0 ? max(max(c, 0) + (nodes - a.window), 0) : 0;
    return c >= 0 && nodes > 0;
}

// Bit b: whether the row sees position p0 + b.
__device__ __forceinline__ uint64_t visible(const PagedAttnArgs& a, const Sight& s, int p0)
{
    const auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };  // bits 0..n - 1
    uint64_t v = below(s.ctx - p0);
    if (a.masks && p0 + 64 > s.ctx && p0 < s.end) {  // not for a column that is none: it has no bits
        const int at = p0 - s.ctx, w = at >> 6, sh = at & 63;  // drafted slot of bit 0, perhaps negative
        const uint64_t lo = w >= 0 && w < a.words ? tree_word(a, s.bits, w) : 0;
        const uint64_t hi = w + 1 >= 0 && w + 1 < a.words ? tree_word(a, s.bits, w + 1) : 0;
        v |= sh ? lo >> sh | hi << (64 - sh) : lo;
    }
    return v & below(s.end - p0) & ~below(s.start - p0);
}

// vector number of head kvh at position p, or -1 where its page is missing
template <bool Q8>
__device__ __forceinline__ long long vector_at(const KvGeom& g, int table, int p, int kvh)
{
    const int b = p / g.tpb;
    const uint32_t blk = g.bt[(size_t)table * g.max_blocks + b];
    if (blk >= (uint32_t)g.total_blocks) return -1;
    const long long page = (long long)blk * g.n_layers + g.layer;
    if constexpr (Q8) return (page * g.n_kv + kvh) * g.tpb + (p - b * g.tpb);
    else return (page * g.tpb + (p - b * g.tpb)) * g.n_kv + kvh;
}

__device__ __forceinline__ float capped(const PagedAttnArgs& a, float s)
{
    return a.cap > 0.0f ? tanhf(s / a.cap) * a.cap : s;
}

// The units of positions lo, lo + step, ... below up of one (row, head) over f16 pages by plain f32 sums, the whole block:
// reference R, log2(e) times the largest score, sum l of the weights and, in threads below HD, the weighted sum of V
// (returned).  A unit at a time: a score per thread, then HD threads per position.  For columns whose sums in f16 parts are not finite: inf * lo may be NaN where
// inf * v is not, and so is the 0 * inf of a position that the column does not see.
template <int HD, int UNIT>
__device__ float plain_range(const PagedAttnArgs& a, const Sight& si, int table, int row, int head, int lo, int up, int step,
                             bool part, unsigned char* lds, float& R, float& l)
{
    long long* const vec = reinterpret_cast<long long*>(lds);
    float* const red = reinterpret_cast<float*>(vec + kThreads);
    float* const ws = red + kThreads;
    const int t = threadIdx.x, kvh = head / (a.n_heads / a.g.n_kv);
    const float* qr = a.q + ((size_t)row * a.n_heads + head) * HD;
    const auto score = [&](long long v) {
        float d = 0.0f;
        const u4_t* src = reinterpret_cast<const u4_t*>(static_cast<const uint16_t*>(a.kc) + v * HD);
#pragma unroll 1
        for (int i = 0; i < HD / 8; ++i) {
            // a missing page counts as zeros, of which an element of q that is not finite makes NaN
            const h8_t w = __builtin_bit_cast(h8_t, v >= 0 ? src[i] : u4_t{0, 0, 0, 0});
#pragma unroll
            for (int j = 0; j < 8; ++j) d = d + qr[8 * i + j] * (float)w[j];
        }
        return capped(a, d * a.scale);
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
    float mt = -INFINITY;
#pragma unroll 1
    for (int p = lo + t; p < up; p += step)
        if (t < UNIT && si.sees(p)) mt = fmaxf(mt, score(vector_at<false>(a.g, table, p, kvh)));
    const float m = reduce(mt, [](float x, float y) { return fmaxf(x, y); });
    R = m * kLog2e;
    constexpr int NP = kThreads / HD;
    const int d = t % HD;
    float lt = 0.0f, o = 0.0f;
#pragma unroll 1
    for (int p0 = lo; p0 < up; p0 += step) {
        const int p = p0 + t;
        long long v = -1;
        float w = 0.0f;
        if (t < UNIT && p < up && si.sees(p)) {
            v = vector_at<false>(a.g, table, p, kvh);
            const float s = score(v);
            // a range whose scores are all -inf weighs nothing beside others, and its l = NaN says that there were some;
            // a NaN among them (m leaves it out) has the weight NaN, which o brings to every split
            w = exp2f(__builtin_fmaf(s, kLog2e, -R));
            lt = lt + w;
            if (part && m == -INFINITY && s == -INFINITY) w = 0.0f;
        }
        __syncthreads();
        vec[t] = v;
        ws[t] = w;
        __syncthreads();
#pragma unroll 1
        for (int j = t / HD; j < min(UNIT, up - p0); j += NP)
            o = o + ws[j] * (vec[j] >= 0 ? (float)static_cast<const _Float16*>(a.vc)[vec[j] * HD + d] : 0.0f);
    }
    l = reduce(lt, [](float x, float y) { return x + y; });
    __syncthreads();
    red[t] = o;
    __syncthreads();
    o = 0.0f;
    if (t < HD)
        for (int j = 0; j < NP; ++j) o = o + red[j * HD + t];
    __syncthreads();
    return o;
}

// Positions lo..hi - 1 that the columns of a set may see; false: none of its rows has a position.
__device__ __forceinline__ bool set_range(const MmaArgs& A, int set, int& lo, int& hi)
{
    const PagedAttnArgs& a = A.a;
    const int table = A.tiles == 1 ? set : set / A.tiles, c0 = (set - table * A.tiles) * A.cols;
    lo = A.cap;
    hi = 0;
    if (a.masks) {
        const int c = a.pos[table], ctx = min(c, A.cap);
        if (c < 0) return false;
        hi = min(ctx + a.per, A.cap);
        lo = a.window > 0 ? min(max(c - a.window + 1, 0), hi - 1) : 0;  // a position at least: rows that see none get zeros
        return true;
    }
    const int j1 = min(a.per - 1, (c0 + A.cols - 1) / A.group);
    for (int j = c0 / A.group; j <= j1; ++j) {
        const int p = a.pos[table * a.per + j];
        if (p < 0) continue;
        const int end = min(p, A.cap - 1) + 1;
        hi = max(hi, end);
        lo = min(lo, a.window > 0 ? max(end - a.window, 0) : 0);
    }
    return hi > 0;
}

struct Work {
    int set, lo, hi, step;      // units of positions lo, lo + step, ... below hi (-1: below the columns' ends)
    int split, splits, slot0;   // slot0: work number of the set's split 0
};

// Work number w of a kv head.  SPLITS: every wave looks at all sets (64 lanes, up to 4 sets each): their positions in units
// of UNIT add up to the work, each set gets as many splits as units, in shares of the same size for all (so that
// contexts of different lengths end together) and at most kMaxSplits, and the splits are numbered through.
template <int UNIT, bool SPLITS>
__device__ __forceinline__ bool plan(const MmaArgs& A, int w, Work& k)
{
    const int lane = threadIdx.x & 63;
    if (!SPLITS || A.want == 0) {
        k = Work{A.sets - 1 - w, 0, -1, UNIT, 0, 1, 0};  // a prompt's last rows, which see the most, first
        if (k.set < 0) return false;
        if (!A.a.masks && A.a.window == 0) return true;  // all from 0 on: how far, the columns will say
        if (!set_range(A, k.set, k.lo, k.hi)) return false;
        k.lo = rfl(k.lo) & ~63;
        k.hi = rfl(k.hi);
        return true;
    }
    constexpr int N = kPlanSets / 64;
    int units[N], from[N], to[N], total = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        units[i] = from[i] = to[i] = 0;
        if (64 * i >= A.sets) continue;  // the same for the whole wave
        const int e = lane + 64 * i;
        if (e < A.sets && set_range(A, e, from[i], to[i])) {
            from[i] &= ~63;
            units[i] = (to[i] - from[i] + UNIT - 1) / UNIT;
        }
        total += units[i];
    }
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    const int share = max(1, (total + A.want - 1) / A.want);
    int base = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (64 * i >= A.sets || found) continue;
        int n = units[i] <= kWholeUnits ? min(units[i], 1) : min(kMaxSplits, (units[i] + share - 1) / share);
        const int each = n > 0 ? (units[i] + n - 1) / n : 1;
        n = (units[i] + each - 1) / each;
        int up = n;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(up, o);
            if (lane >= o) up += v;
        }
        const int first = base + up - n;
        const unsigned long long hit = __ballot(w >= first && w < first + n);
        if (hit) {  // one lane
            const int src = __builtin_ctzll(hit);
            found = true;
            k.set = src + 64 * i;
            k.splits = __builtin_amdgcn_readlane(n, src);
            k.slot0 = __builtin_amdgcn_readlane(first, src);
            k.split = w - k.slot0;
            k.lo = __builtin_amdgcn_readlane(from[i], src) + k.split * UNIT;
            k.hi = __builtin_amdgcn_readlane(to[i], src);
            k.step = k.splits * UNIT;
        }
        base += __builtin_amdgcn_readlane(up, 63);
    }
    return found;
}

template <bool Q8, int HD, int CT = 1>
struct Shape {
    static constexpr int CH = Q8 ? (HD == 64 || (HD == 128 && CT == 1) ? 64 : 32) : HD == 64 ? 64 : 32;  // positions of a chunk
    static constexpr int ES = Q8 ? 1 : 2;                    // bytes of an element of K and V
    static constexpr int KK = Q8 ? HD / 64 : HD / 32;        // k steps of a K tile
    static constexpr int QP = Q8 ? 3 : 2;                    // parts of q
    static constexpr int NE = Q8 ? 16 : 8;                   // elements of q of a lane and k step: NE (4 kk + g) + 0, 1, ...
    static constexpr int DT = HD / 16;                       // tiles of O^T
};

// Codes of four dims at positions j (a) and j + 1 (b) as f16 pairs by dim, in units of 2^-9, all exact: the byte c + 128
// alone is the f16 (c + 128) 2^-24, and (c + 128) 2^-24 * 2^15 - 2^-2 = c 2^-9.
constexpr float kCodeUnit = 0x1p9f;
__device__ __forceinline__ void pairs_of_codes(uint32_t a, uint32_t b, uint32_t (&o)[4])
{
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const h2_t up = {(_Float16)0x1p15f, (_Float16)0x1p15f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
    o[0] = as_u32(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(b, a, 0x0C040C00u)), up, off));
    o[1] = as_u32(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(b, a, 0x0C050C01u)), up, off));
    o[2] = as_u32(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(b, a, 0x0C060C02u)), up, off));
    o[3] = as_u32(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(b, a, 0x0C070C03u)), up, off));
}

// The sums of q's integers reach 2^37, so scales of keys near the end of f32 would take them past it before the scale of a
// tiny q brings them back: in a chunk that has a scale above kHugeKey all are taken 2^kHugeShift times smaller, and the
// column's scale as much larger.
constexpr float kHugeKey = 0x1p80f;
constexpr int kHugeShift = 40;

// Three digits leave every element a rounding of 2^-23 of the largest, f32 one of 2^-25 of itself, beside sums that cost
// some 2^-24: heads whose largest |q| is more than kLoud times the mean |q| take the fourth digit (normally distributed
// elements have 3 to 5 times).  Error of the output with one element 30 and 300 times the others, where the keys hold
// zeros: 3.5e-6 and 3.1e-5 with three digits, 4.2e-7 and 4.6e-7 with four (all f32: 2e-7).  Time, 8 sessions at 8192
// positions, 32/8 heads of 128, and a prompt of 1024: 28.8 and 84.0 us without the digit, 29.3 and 84.9 with the test for
// it in each chunk, 31.2 and 92.4 where it is taken.
constexpr float kLoud = 8.0f;

// q's parts of a column, the B operands of the scores, and the scale that is left out of them: for scales of the keys as
// they are and, of 8-bit pages, for those of a chunk with huge ones (kHugeKey).  8-bit pages: the fourth digits, and
// whether some column of the wave needs them.
template <bool Q8, int HD>
__device__ __forceinline__ void q_parts(const PagedAttnArgs& a, const f4_t (&qf)[Shape<Q8, HD>::KK][Shape<Q8, HD>::NE / 4],
                                        u4_t (&d)[Shape<Q8, HD>::KK][Shape<Q8, HD>::QP], u4_t (&low)[Shape<Q8, HD>::KK],
                                        bool& loud, float (&qsc)[2])
{
    using S = Shape<Q8, HD>;
    uint32_t mx = 0;  // |q| in the order of its bits; f16 pages: of the finite ones
    float sum = 0.0f;
#pragma unroll
    for (int kk = 0; kk < S::KK; ++kk)
#pragma unroll
        for (int i = 0; i < S::NE; ++i) {
            const float x = qf[kk][i >> 2][i & 3];  // a bit_cast of the element itself reads the vector's first
            const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu;
            mx = max(mx, Q8 || b < 0x7F800000u ? b : 0u);
            if constexpr (Q8) sum = sum + fabsf(x);
        }
    mx = max(mx, __builtin_bit_cast(uint32_t, lane_xor<16>(__builtin_bit_cast(float, mx), 64)));
    mx = max(mx, __builtin_bit_cast(uint32_t, lane_xor<32>(__builtin_bit_cast(float, mx), 64)));
    const int top = max((int)(mx >> 23), 1) - 127;
    const bool bad = Q8 && mx >= 0x7F800000u;
    const int e = mx > 0 && !bad ? (Q8 ? 21 : 13) - top : 0;
    qsc[0] = bad ? __builtin_nanf("") : ldexpf(a.scale, -e);
    qsc[1] = Q8 ? (bad ? __builtin_nanf("") : ldexpf(a.scale, kHugeShift - e)) : 0.0f;
#pragma unroll
    for (int kk = 0; kk < S::KK; ++kk) {
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the four bytes less 128 are the balanced digits
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (uint32_t)(int)rintf(bad ? 0.0f : ldexpf(qf[kk][i][j], e + 8)) + 0x80808080u;
                const uint32_t a01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), a23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
                const uint32_t b01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), b23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
                low[kk][i] = __builtin_amdgcn_perm(a23, a01, 0x05040100u) ^ 0x80808080u;
                d[kk][0][i] = __builtin_amdgcn_perm(a23, a01, 0x07060302u) ^ 0x80808080u;
                d[kk][1][i] = __builtin_amdgcn_perm(b23, b01, 0x05040100u) ^ 0x80808080u;
                d[kk][2][i] = __builtin_amdgcn_perm(b23, b01, 0x07060302u) ^ 0x80808080u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h2_t hi, lo;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int x = 2 * i + j;
                    const float v = ldexpf(qf[kk][x >> 2][x & 3], e);
                    hi[j] = (_Float16)v;
                    lo[j] = finite_f32(v) ? (_Float16)(v - (float)hi[j]) : (_Float16)0.0f;
                }
                d[kk][0][i] = as_u32(hi);
                d[kk][1][i] = as_u32(lo);
            }
        }
    }
    if constexpr (Q8) {
        sum = sum + lane_xor<16>(sum, 64);
        sum = sum + lane_xor<32>(sum, 64);
        loud = __ballot(!bad && sum / HD < __builtin_bit_cast(float, mx) / kLoud) != 0;  // a sum past f32 is none
    }
}

// A column's sums so far: reference (the first chunk's weights pass any bound), sum of the weights, O^T in units of 1 / F.
template <int DT>
struct Sums {
    float R, l, F;
    f4_t o[DT];
};

// Scores s of NP positions (bit 4 j of vis: position j is seen; `partial`: not all are, in some column) and their scales
// vs to the weights' two f16 parts, and into l; the reference is raised where products pass 2^15 (or weights 2^80).
template <bool Q8, int NP, int DT>
__device__ __forceinline__ void weigh(const float (&s)[NP], float cs, const float (&vs)[NP], bool partial, uint64_t vis, bool& coarse,
                                      Sums<DT>& m, h8_t (&ph)[NP / 8], h8_t (&pl)[NP / 8])
{
    float w[NP], lc, mx;
    const auto weights = [&]() {
        lc = mx = 0.0f;
#pragma unroll
        for (int j = 0; j < NP; ++j) w[j] = __builtin_amdgcn_exp2f(s[j] * cs - m.R);
        if (partial) {
            asm volatile("");  // a branch
#pragma unroll
            for (int j = 0; j < NP; ++j) w[j] = vis >> (4 * j) & 1 ? w[j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            lc = lc + w[j];
            if constexpr (Q8) w[j] = w[j] * vs[j];
            mx = fmaxf(mx, w[j]);
        }
        if (Q8 && coarse) {
            asm volatile("");
            mx = mx * m.F;
#pragma unroll
            for (int j = 0; j < NP; ++j) w[j] = w[j] * m.F;
        }
    };
    weights();
    if (__ballot(mx > 0x1p15f || lc > 0x1p80f)) {
        // The reference that leaves the largest product at 2^13.  8-bit pages: not so far from the largest score that a
        // sum of weights under another reference (of another wave or split, or this one so far) would leave f32 beside
        // it; what the scales of the values then miss of 2^13, and what a reference beyond 2^20 has no bits for, F makes up.
        float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const float h = vis >> (4 * j) & 1 ? s[j] * cs : -INFINITY;
            m1 = fmaxf(m1, h);
            if constexpr (Q8) m2 = fmaxf(m2, h + __builtin_amdgcn_logf(vs[j]));
        }
        m1 = fmaxf(m1, lane_xor<16>(m1, 64));
        m1 = fmaxf(m1, lane_xor<32>(m1, 64));
        if constexpr (Q8) {
            m2 = fmaxf(m2, lane_xor<16>(m2, 64));
            m2 = fmaxf(m2, lane_xor<32>(m2, 64));
        }
        const float up = fmaxf(m.R, Q8 ? fminf(fmaxf(m2 - 13.0f, m1 - 60.0f), m1 + 30.0f) : m1 - 13.0f);
        float ratio = up > m.R ? __builtin_amdgcn_exp2f(m.R - up) : 1.0f;  // from -inf: 0, as l and O are
        m.l = m.l * ratio;
        if constexpr (Q8) {
            const float over = m2 - up;  // the largest product; NaN: nothing is seen here, nor was before
            if (coarse || __ballot(over > 15.0f || (up > m.R && over < 12.0f))) {
                if (over < 1000.0f) {
                    const float want = __builtin_amdgcn_exp2f(fminf(fmaxf(13.0f - rintf(over), -100.0f), 100.0f));
                    // up by as much as R rose at most: what O holds is not to pass its bound
                    const float most = up > m.R ? m.F * __builtin_amdgcn_exp2f(up - m.R) : m.F;
                    const float f = m.F > 4.0f * want ? want : fminf(fmaxf(m.F, want), most);
                    if (ratio > 0.0f) ratio = ratio * (f / m.F);
                    m.F = f;
                }
                coarse = coarse || __ballot(m.F != 1.0f) != 0;
            }
        }
        m.R = up;
#pragma unroll
        for (int e = 0; e < DT; ++e) m.o[e] = m.o[e] * ratio;
        weights();
    }
    m.l = m.l + lc;
    // w - h, exact in f32, and its rounding to f16 are one instruction where the compiler sees a product
    float minus1 = -1.0f;
    asm("" : "+s"(minus1));
#pragma unroll
    for (int j = 0; j < NP; j += 2) {
        const h2_t h = {(_Float16)w[j], (_Float16)w[j + 1]};
        const h2_t l = {(_Float16)__builtin_fmaf((float)h[0], minus1, w[j]), (_Float16)__builtin_fmaf((float)h[1], minus1, w[j + 1])};
        ph[j >> 3][j & 7] = h[0];
        ph[j >> 3][(j & 7) + 1] = h[1];
        pl[j >> 3][j & 7] = l[0];
        pl[j >> 3][(j & 7) + 1] = l[1];
    }
}

// Words of four (8-bit) or two (f16) dims at eight positions as the V^T operands of those dims
template <bool Q8>
__device__ __forceinline__ void v_operands(const uint32_t (&r)[8], u4_t (&vt)[Q8 ? 4 : 2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Q8) {
            uint32_t y[4];
            pairs_of_codes(r[2 * i], r[2 * i + 1], y);
#pragma unroll
            for (int e = 0; e < 4; ++e) vt[e][i] = y[e];
        } else {
            vt[0][i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x05040100u);
            vt[1][i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x07060302u);
        }
    }
}

// scores of a tile's 16 positions from the sums of q's parts
__device__ __forceinline__ float score_of(int hi, int mid, int lo, float ks)
{
    return __builtin_fmaf((float)hi, 65536.0f, (float)(mid * 256 + lo)) * ks;
}

// ---- a block's results: its sums where the set is split, else the quotients; the sums of splits added by the last ----
// COLS columns of a set from column col0 of the table on; a split's sums: [COLS][HD], then R and l, [COLS] each.  Sets of
// 32 columns are taken where they leave kWideBlocks blocks, and split where there are fewer than kPlanBlocks: never.
template <int HD, int COLS>
struct Results {
    static constexpr bool kSplits = COLS == kCols;
    static_assert(kSplits || kWideBlocks >= kPlanBlocks);
    static constexpr uint32_t kPart = COLS * (HD + 2);
    const MmaArgs& A;
    const Work& k;
    int table, col0, kvh;
    __amdgpu_buffer_rsrc_t part;
    __device__ __forceinline__ Results(const MmaArgs& A_, const Work& k_, int kvh_)
        : A(A_), k(k_), table(A_.tiles == 1 ? k_.set : k_.set / A_.tiles), col0((k_.set - table * A_.tiles) * COLS), kvh(kvh_), part(buffer_rsrc(A_.part, A_.part_bytes))
    {
    }
    __device__ __forceinline__ int columns() const { return min(A.a.per * A.group - col0, COLS); }
    struct Column {
        int row, head;
    };
    __device__ __forceinline__ Column column(int x) const
    {
        const int j = (col0 + x) / A.group;
        return {table * A.a.per + j, kvh * A.group + (col0 + x) - j * A.group};
    }
    __device__ __forceinline__ size_t offset(Column c) const { return ((size_t)c.row * A.a.n_heads + c.head) * HD; }  // in q and out
    __device__ __forceinline__ uint32_t part_of(int sp) const { return (uint32_t)((k.slot0 + sp) * A.a.g.n_kv + kvh) * kPart; }
    // four dims of column x (at offset `at` of out) from d on, ll the sum of all its weights; whether they are finite
    __device__ __forceinline__ bool put(int x, size_t at, int d, f4_t v, float ll) const
    {
        if (kSplits && k.splits > 1) st_agent4(part, part_of(k.split) + x * HD + d, v);
        else *reinterpret_cast<f4_t*>(A.a.out + at + d) = v * (ll != 0.0f ? 1.0f / ll : 0.0f);
        return finite_f32(v[0]) && finite_f32(v[1]) && finite_f32(v[2]) && finite_f32(v[3]) && finite_f32(ll);
    }
    __device__ __forceinline__ void put_sums(int x, float r, float ll) const
    {
        st_agent(part, part_of(k.split) + COLS * HD + x, r);
        st_agent(part, part_of(k.split) + COLS * (HD + 1) + x, ll);
    }
    // f16 pages: the columns whose bits `again` has by plain sums; the whole block
    template <int UNIT>
    __device__ void put_plain(uint32_t again, unsigned char* lds) const
    {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // their first values are written
        __syncthreads();
#pragma unroll 1
        for (int x = 0; x < COLS; ++x) {
            if (!(again >> x & 1)) continue;
            const Column c = column(x);
            Sight sc;
            sight_of(A.a, A.cap, table, c.row, sc);
            float mm, ll;
            const float v = plain_range<HD, UNIT>(A.a, sc, table, c.row, c.head, k.lo, sc.end, k.step, kSplits && k.splits > 1, lds, mm, ll);
            const int t = threadIdx.x;
            if (kSplits && k.splits > 1) {
                if (t < HD) st_agent(part, part_of(k.split) + x * HD + t, v);
                if (t == 0) put_sums(x, mm, ll);
            } else if (t < HD) {
                A.a.out[offset(c) + t] = ll != 0.0f ? v / ll : 0.0f;
            }
        }
    }
    // The last block of a split set to get here adds the splits; bit x of `here`: column x is there; lds: COLS * kMaxSplits * 8
    // bytes, half of them at least 16 a thread.
    __device__ void combine(const uint32_t& here, float* lsum, int* last, unsigned char* lds) const
    {
        const int t = threadIdx.x, lane = t & 63, wave = rfl(t >> 6), n = k.splits;
        if (n <= 1) return;
        // this block's sums are performed at the coherence point before it counts itself
        uint32_t* const counter = A.counters + (size_t)k.set * A.a.g.n_kv + kvh;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t == 0)
            *last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(n - 1);
        __syncthreads();
        if (!*last) return;
        // The splits' references and sums of weights to LDS, then weights 2^(R_k - R).  The values: an item is four dims
        // of a column; few items share their splits among groups of threads, which meet in LDS.
        float* const mk = reinterpret_cast<float*>(lds);  // [column][kMaxSplits], then the weights
        float* const lk = mk + COLS * kMaxSplits;
        f4_t* const red = reinterpret_cast<f4_t*>(lk);    // once lk is read
        const uint32_t present = here;
        const auto there = [&](int x) { return present >> x & 1; };
        const int cols = columns(), items = cols * (HD / 4), groups = max(1, kThreads / items);
        constexpr int U = 8;  // loads in flight
        f4_t v[U];
        const int group = t / items;
        int item = t - group * items;
        bool busy = group < groups && t < groups * items;
        const auto load = [&](int sp) {
#pragma unroll
            for (int j = 0; j < U; ++j) v[j] = ld_agent4(part, part_of(min(sp + j * groups, n - 1)) + 4 * item);
        };
        if (busy) load(group);
        for (int i = t; i < COLS * n; i += kThreads) {
            const int sp = i / COLS, x = i % COLS;
            if (!there(x)) continue;
            mk[x * kMaxSplits + sp] = ld_agent(part, part_of(sp) + COLS * HD + x);
            lk[x * kMaxSplits + sp] = ld_agent(part, part_of(sp) + COLS * (HD + 1) + x);
        }
        __syncthreads();
        for (int x = wave; x < cols; x += kWaves) {
            if (!there(x)) continue;
            const float mv = lane < n ? mk[x * kMaxSplits + lane] : -INFINITY, lv = lane < n ? lk[x * kMaxSplits + lane] : 0.0f;
            const float mm = group_max<64>(mv);
            // a split without a score above -inf weighs nothing beside others; where all are so, its l is 0 (nothing
            // seen: zeros) or NaN
            const float ew = mv > -INFINITY ? __builtin_amdgcn_exp2f(mv - mm) : mm > -INFINITY ? 0.0f : 1.0f;
            const float ll = group_sum<64>(mv > -INFINITY || !(mm > -INFINITY) ? lv * ew : 0.0f);
            if (lane < n) mk[x * kMaxSplits + lane] = ew;
            if (lane == 0) lsum[x] = ll;
        }
        __syncthreads();
        for (;;) {  // more than 256 items: again for the others, in one group
            f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
            const int x = min(item / (HD / 4), COLS - 1);
            if (busy) {
                for (int sp = group; sp < n; sp += U * groups) {
                    if (sp > group) load(sp);
#pragma unroll
                    for (int j = 0; j < U; ++j)
                        if (sp + j * groups < n) acc = acc + v[j] * mk[x * kMaxSplits + sp + j * groups];
                }
            }
            if (groups > 1) {
                red[t] = acc;
                __syncthreads();
                if (group == 0)
                    for (int y = 1; y < groups; ++y) acc = acc + red[y * items + t];
            }
            if (busy && group == 0 && there(x)) {
                const float ll = lsum[x];
                *reinterpret_cast<f4_t*>(A.a.out + offset(column(x)) + 4 * (item % (HD / 4))) = acc * (ll != 0.0f ? 1.0f / ll : 0.0f);
            }
            item += kThreads;
            if (groups > 1 || item - t >= items) break;
            busy = item < items;
            if (busy) load(0);
        }
        if (t == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
};

// One set of 16 CT columns a block; its waves take chunks of the positions in turn and meet in LDS.
template <bool Q8, int HD, int CT, bool CAP>
__global__ __launch_bounds__(kThreads, 2) void attn_paged_kernel(const MmaArgs A)
{
    using S = Shape<Q8, HD, CT>;
    constexpr int CH = S::CH, NT = CH / 16, NP = CH / 4, KS = CH / 32;  // K tiles; positions of a lane; k steps of V
    constexpr int KK = S::KK, QP = S::QP, NE = S::NE, DT = S::DT, VW = DT * S::ES / 4;  // VW: words of V per lane and position
    constexpr int NR = HD / 4 < 32 ? HD / 4 : 32;                       // registers of O^T that the waves add at a time
    constexpr bool kQInLds = HD > 128 || CT > 1;                        // q's parts in LDS, for want of registers
    constexpr int COLS = kCols * CT;
    constexpr bool kSplits = Results<HD, COLS>::kSplits;
    constexpr int kMergeBytes = std::max(kWaves * NR * 64 * 4, kSplits ? COLS * kMaxSplits * 8 : 0);
    __shared__ __align__(16) unsigned char merge[kMergeBytes];
    __shared__ __align__(16) u4_t qlds[kQInLds ? CT * KK * QP * 64 : 1];
    __shared__ __align__(16) u4_t qlow[Q8 ? CT * KK * 64 : 1];          // the fourth digits
    __shared__ uint32_t loud_lds[CT];
    __shared__ __align__(16) uint32_t kidx[kWaves][CH], vidx[kWaves][CH];  // [c][tile], [g][j]
    __shared__ __align__(16) float kscl[kWaves][Q8 ? CH : 4], vscl[kWaves][Q8 ? CH : 4];
    __shared__ float ml[kWaves][2][COLS], lsum[kSplits ? COLS : 1], qs_lds[2][COLS];
    __shared__ uint32_t flags, here;
    __shared__ int last;

    const PagedAttnArgs& a = A.a;
    const int t = threadIdx.x, lane = t & 63, wave = rfl(t >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    const int kvh = blockIdx.x;
    Work k;
    if (!plan<kWaves * CH, kSplits>(A, blockIdx.y + gridDim.y * blockIdx.z, k)) return;  // the same for the whole block
    const Results<HD, COLS> res(A, k, kvh);
    const int table = res.table, n_cols = res.columns();

    // ---- the first chunk's page entries, q, and what this lane's column sees: loads that do not wait for each other
    const auto block_of = [&](int p) { return A.tpb_shift >= 0 ? p >> A.tpb_shift : p / a.g.tpb; };
    const uint32_t* const bt = a.g.bt + (size_t)table * a.g.max_blocks;
    int p0 = k.lo + wave * CH;
    const int b_first = block_of(p0 + (lane & (CH - 1)));
    const uint32_t blk_first = bt[min(b_first, a.g.max_blocks - 1)];
    Sight si[CT];
    bool has[CT];
    size_t at[CT];             // of the column in q and out
    u4_t qp[CT][KK][QP];
    float qsc[CT][2];          // scale of the sums of q's parts
    bool loud = false;         // some column needs the fourth digits
    Sums<DT> m[CT];
    // with q's parts in LDS wave u makes those of the columns 16 u + c
    const auto makes = [&](int u) { return !kQInLds || wave == u; };
    {
        f4_t qf[CT][KK][NE / 4];
        uint32_t b = 0;
        int top = 0;
#pragma unroll
        for (int u = 0; u < CT; ++u) {
            const auto x = res.column(min(kCols * u + c, n_cols - 1));
            at[u] = res.offset(x);
            if (makes(u)) {
                const f4_t* src = reinterpret_cast<const f4_t*>(a.q + at[u] + NE * g4);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                    for (int i = 0; i < NE / 4; ++i) qf[u][kk][i] = src[NE * kk + i];
            }
            si[u] = Sight{0, 0, 0, a.masks};
            has[u] = sight_of(a, A.cap, table, x.row, si[u]) && kCols * u + c < n_cols;
            if (!has[u]) si[u] = Sight{0, 0, 0, a.masks};
            b |= ((uint32_t)__ballot(has[u]) & 0xFFFFu) << (kCols * u);
            top = max(top, si[u].end);
            m[u] = Sums<DT>{-INFINITY, 0.0f, 1.0f, {}};
        }
        if (k.hi < 0) k.hi = rfl((int)team_max_u32<16>((uint32_t)top));
        if (t == 0) {
            here = b;
            flags = 0;
        }
#pragma unroll
        for (int u = 0; u < CT; ++u) {
            if (!makes(u)) continue;
            u4_t low[KK];
            q_parts<Q8, HD>(a, qf[u], qp[u], low, loud, qsc[u]);
            if (Q8 && (kQInLds || (loud && wave == 0))) {
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) qlow[(u * KK + kk) * 64 + lane] = low[kk];
            }
            if constexpr (kQInLds) {
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                    for (int p = 0; p < QP; ++p) qlds[((u * KK + kk) * QP + p) * 64 + lane] = qp[u][kk][p];
                if (g4 == 0) {
                    qs_lds[0][kCols * u + c] = qsc[u][0];
                    qs_lds[1][kCols * u + c] = qsc[u][1];
                }
                if (Q8 && lane == 0) loud_lds[u] = loud;
            }
        }
        if constexpr (kQInLds) {
            __syncthreads();
            loud = false;
#pragma unroll
            for (int u = 0; u < CT; ++u) {
                qsc[u][0] = qs_lds[0][kCols * u + c];
                qsc[u][1] = qs_lds[1][kCols * u + c];
                if (Q8) loud = loud || rfl((int)loud_lds[u]) != 0;
            }
        } else if (Q8 && loud) {
            __syncthreads();  // the same for all waves, whose columns are the same
        }
        if constexpr (!CAP) {  // and of the exponents
#pragma unroll
            for (int u = 0; u < CT; ++u) {
                qsc[u][0] = qsc[u][0] * kLog2e;
                qsc[u][1] = qsc[u][1] * kLog2e;
            }
        }
    }
    const auto q_part = [&](int u, int p, int kk) {
        if constexpr (kQInLds) return qlds[((u * KK + kk) * QP + p) * 64 + lane];
        else return qp[u][kk][p];
    };
    bool coarse = false;  // F is not 1 somewhere
    const unsigned char* const kbase = static_cast<const unsigned char*>(a.kc) + 16 * g4;
    const unsigned char* const vbase = static_cast<const unsigned char*>(a.vc) + DT * S::ES * c;

    // A chunk's loads are issued an iteration ahead, into the registers that its predecessor has just used: K and the
    // scales after the scores, V after the weighted sums, page entries two chunks ahead.  The last iteration loads too:
    // behind a branch every wait for V would be one for the K issued after it.
    uint32_t blk;                       // page entry of this lane's position, of the chunk whose indexes come next
    int b_of;                           // its place in the table
    unsigned long long miss, miss_next; // positions without a page, or past the range
    float ks_own = 0.0f, vs_own = 0.0f;
    u4_t kr[NT][KK];
    uint32_t vr[NP][VW];
    uint32_t vn = 0;
    const auto load_page = [&](int p0) {
        b_of = block_of(p0 + (lane & (CH - 1)));
        blk = bt[min(b_of, a.g.max_blocks - 1)];
    };
    const auto index = [&](int p0) {    // vector numbers of the chunk at p0 into LDS
        const int pp = p0 + (lane & (CH - 1));
        const bool ok = pp < k.hi && b_of < a.g.max_blocks && blk < (uint32_t)a.g.total_blocks;
        const uint32_t page = blk * (uint32_t)a.g.n_layers + (uint32_t)a.g.layer, off = (uint32_t)(pp - b_of * a.g.tpb);
        // where there is none: the last vector again, loaded but not used
        vn = !ok ? vn : Q8 ? (page * (uint32_t)a.g.n_kv + (uint32_t)kvh) * (uint32_t)a.g.tpb + off
                           : (page * (uint32_t)a.g.tpb + off) * (uint32_t)a.g.n_kv + (uint32_t)kvh;
        miss_next = __ballot(!ok);
        wave_lds_fence();
        if (lane < CH) {  // position 16 tile + 4 i + g
            const int tile = lane >> 4, i = lane >> 2 & 3, g = lane & 3;
            kidx[wave][(4 * g + i) * NT + tile] = vn;
            vidx[wave][g * NP + 4 * tile + i] = vn;
        }
        wave_lds_fence();
    };
    const auto load_k = [&]() {
        if constexpr (Q8) {
            ks_own = a.ks[vn];
            vs_own = a.vs[vn];
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const unsigned char* src = kbase + (size_t)kidx[wave][c * NT + i] * (HD * S::ES);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) kr[i][kk] = *reinterpret_cast<const u4_t*>(src + 64 * kk);
        }
        asm volatile("" ::: "memory");  // issued here
    };
    const auto load_v = [&]() {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const unsigned char* src = vbase + (size_t)vidx[wave][g4 * NP + j] * (HD * S::ES);
            if constexpr (VW == 1) vr[j][0] = *reinterpret_cast<const uint32_t*>(src);
            else if constexpr (VW == 2) {
                const u2_t v = *reinterpret_cast<const u2_t*>(src);
                vr[j][0] = v[0];
                vr[j][1] = v[1];
            } else {
#pragma unroll
                for (int w = 0; w < VW / 4; ++w) {
                    const u4_t v = *reinterpret_cast<const u4_t*>(src + 16 * w);
#pragma unroll
                    for (int x = 0; x < 4; ++x) vr[j][4 * w + x] = v[x];
                }
            }
        }
        asm volatile("" ::: "memory");
    };
    const int step = k.step;
    if (p0 < k.hi) {
        b_of = b_first;
        blk = blk_first;
        index(p0);
        load_page(p0 + step);
        load_k();
        load_v();
    }
    for (; p0 < k.hi; p0 += step) {
        miss = miss_next;
        bool huge = false;
        if constexpr (Q8) {
            huge = __ballot(ks_own > kHugeKey) != 0;
            if (huge) ks_own = ldexpf(ks_own, -kHugeShift);
            if (lane < CH) {
                const int tile = lane >> 4, i = lane >> 2 & 3, g = lane & 3;
                const bool gone = miss >> lane & 1;  // a missing page counts as zeros
                kscl[wave][g * NP + 4 * tile + i] = gone ? 0.0f : ks_own;
                vscl[wave][g * NP + 4 * tile + i] = gone ? 0.0f : vs_own;
            }
        }
        index(p0 + step);
        load_page(p0 + 2 * step);
        if (!Q8 && miss) {  // a missing page counts as zeros, and so do the positions past the range
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const bool gone = miss >> (16 * i + 4 * (c & 3) + (c >> 2)) & 1;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) kr[i][kk] = gone ? u4_t{0, 0, 0, 0} : kr[i][kk];
            }
        }
        h8_t ph[CT][KS], pl[CT][KS];
#pragma unroll
        for (int u = 0; u < CT; ++u) {
            // ---- scores of positions p0 + 4 j + g4, less their scale qsc without a cap
            float s[NP];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if constexpr (Q8) {
                    i4_t d[3] = {};
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                        for (int p = 0; p < 3; ++p)
                            d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4_t, kr[i][kk]),
                                                                         __builtin_bit_cast(i4_t, q_part(u, p, kk)), d[p], 0, 0, 0);
                    const f4_t ksv = *reinterpret_cast<const f4_t*>(&kscl[wave][g4 * NP + 4 * i]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[4 * i + x] = score_of(d[2][x], d[1][x], d[0][x], ksv[x]);
                } else {
                    f4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = 1; p >= 0; --p)  // the low parts first
#pragma unroll
                        for (int kk = 0; kk < KK; ++kk)
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, kr[i][kk]),
                                                                       __builtin_bit_cast(h8_t, q_part(u, p, kk)), d, 0, 0, 0);
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[4 * i + x] = d[x];
                }
            }
            if (Q8 && loud) {
                asm volatile("");  // a branch
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    i4_t d = {};
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk)
                        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4_t, kr[i][kk]),
                                                                  __builtin_bit_cast(i4_t, qlow[(u * KK + kk) * 64 + lane]), d, 0, 0, 0);
                    const f4_t ksv = *reinterpret_cast<const f4_t*>(&kscl[wave][g4 * NP + 4 * i]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[4 * i + x] = s[4 * i + x] + (float)d[x] * 0x1p-8f * ksv[x];
                }
            }
            if (u == CT - 1) load_k();
            float cs = huge ? qsc[u][1] : qsc[u][0];
            if constexpr (CAP) {
#pragma unroll
                for (int j = 0; j < NP; ++j) s[j] = capped(a, s[j] * cs);
                cs = kLog2e;
            }
            // ---- weights; of positions that some column does not see, those are 0 whatever they hold
            float vs[NP];
#pragma unroll
            for (int j = 0; j < NP; ++j) vs[j] = Q8 ? vscl[wave][g4 * NP + j] : 1.0f;
            const bool partial = __ballot(has[u] && (p0 < si[u].start || p0 + CH > si[u].ctx)) != 0;
            uint64_t vis = ~0ull;  // bit 4 j: position j of this lane
            if (partial) {
                vis = visible(a, si[u], p0) >> g4;
#pragma unroll
                for (int j = 0; j < NP; ++j) vs[j] = vis >> (4 * j) & 1 ? vs[j] : 0.0f;
            }
            weigh<Q8>(s, cs, vs, partial, vis, coarse, m[u], ph[u], pl[u]);
        }
        // ---- O^T += V^T . P^T
        if (!Q8 && miss) {
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int x = 0; x < VW; ++x) vr[j][x] = miss >> (4 * j + g4) & 1 ? 0u : vr[j][x];
        }
#pragma unroll
        for (int x = 0; x < VW; ++x)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                constexpr int E = Q8 ? 4 : 2;  // tiles of a word
                uint32_t r[8];
                u4_t vt[E];
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j] = vr[8 * ks + j][x];
                v_operands<Q8>(r, vt);
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int u = 0; u < CT; ++u) {
                        const h8_t v = __builtin_bit_cast(h8_t, vt[e]);
                        f4_t& o = m[u].o[E * x + e];
                        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[u][ks], o, 0, 0, 0);
                        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[u][ks], o, 0, 0, 0);
                    }
            }
        load_v();
    }

    // ---- the waves meet: each adds a quarter of the registers over all four; lane (c, g) holds dims g HD / 4 + r of its
    // column, r = 0..HD / 4 - 1, in register (r % DT, r / DT)
    float* const mine = reinterpret_cast<float*>(merge) + lane;
    bool fine[CT];
#pragma unroll
    for (int u = 0; u < CT; ++u) {
        const int col = kCols * u + c;
        m[u].l = m[u].l + lane_xor<16>(m[u].l, 64);
        m[u].l = m[u].l + lane_xor<32>(m[u].l, 64);
        if (Q8 && coarse) {
#pragma unroll
            for (int e = 0; e < DT; ++e) m[u].o[e] = m[u].o[e] / m[u].F;
        }
        if (g4 == 0) {
            ml[wave][0][col] = m[u].R;
            ml[wave][1][col] = m[u].l;
        }
        fine[u] = true;
#pragma unroll
        for (int rd = 0; rd < HD / 4 / NR; ++rd) {
            if (u || rd) __syncthreads();
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int x = rd * NR + r;
                mine[(wave * NR + r) * 64] = m[u].o[x % DT][x / DT];
            }
            __syncthreads();
            float mm = ml[0][0][col], ll = 0.0f, acc[NR / 4];
#pragma unroll
            for (int x = 1; x < kWaves; ++x) mm = fmaxf(mm, ml[x][0][col]);
#pragma unroll
            for (int r = 0; r < NR / 4; ++r) acc[r] = 0.0f;
#pragma unroll
            for (int x = 0; x < kWaves; ++x) {
                // no weight (l is 0, or NaN)
                const float ew = ml[x][0][col] > -INFINITY ? __builtin_amdgcn_exp2f(ml[x][0][col] - mm) : ml[x][1][col];
                ll = ll + ml[x][1][col] * ew;
#pragma unroll
                for (int r = 0; r < NR / 4; ++r) acc[r] = acc[r] + mine[(x * NR + wave * (NR / 4) + r) * 64] * (Q8 ? ew * kCodeUnit : ew);
            }
            if (has[u]) {
#pragma unroll
                for (int r = 0; r < NR / 4; r += 4)
                    fine[u] &= res.put(col, at[u], g4 * (HD / 4) + rd * NR + wave * (NR / 4) + r,
                                       f4_t{acc[r], acc[r + 1], acc[r + 2], acc[r + 3]}, ll);
                if (kSplits && k.splits > 1 && rd == 0 && wave == 0 && g4 == 0) res.put_sums(col, mm, ll);
            }
        }
    }
    if constexpr (!Q8) {
#pragma unroll
        for (int u = 0; u < CT; ++u)
            if (!fine[u]) atomicOr(&flags, 1u << (kCols * u + c));
        __syncthreads();
        const uint32_t again = flags;
        if (again) res.template put_plain<kWaves * CH>(again, merge);  // rare
    }
    if constexpr (kSplits) res.combine(here, lsum, &last, merge);
}

template <typename F>
void by_shape(bool q8, int head_dim, F&& f)
{
    const auto with = [&](auto q) {
        if (head_dim == 64) f(q, std::integral_constant<int, 64>{});
        else if (head_dim == 128) f(q, std::integral_constant<int, 128>{});
        else f(q, std::integral_constant<int, 256>{});
    };
    q8 ? with(std::true_type{}) : with(std::false_type{});
}

struct Layout {
    int ct, group, cols, tiles, sets, want;
    long long works;  // per kv head
};

Layout layout_of(const PagedAttnArgs& a)
{
    Layout y{};
    y.group = a.n_heads / a.g.n_kv;
    const long long columns = (long long)a.per * y.group, tables = a.rows / a.per;
    y.ct = a.head_dim <= 128 && columns > kCols && tables * a.g.n_kv * ((columns + 31) / 32) >= kWideBlocks ? 2 : 1;
    y.cols = kCols * y.ct;
    y.tiles = (int)((columns + y.cols - 1) / y.cols);
    y.sets = (int)(tables * y.tiles);
    int unit = 0;
    by_shape(a.ks != nullptr, a.head_dim,
             [&](auto q, auto hd) {
                 constexpr bool Q8 = decltype(q)::value;
                 constexpr int HD = decltype(hd)::value;
                 unit = (y.ct == 2 ? Shape<Q8, HD, 2>::CH : Shape<Q8, HD>::CH) * kWaves;
             });
    const long long cap = (long long)a.g.max_blocks * a.g.tpb, units = (cap + unit - 1) / unit;
    const long long blocks = (long long)y.sets * a.g.n_kv;
    if (blocks < kPlanBlocks && units > kWholeUnits) y.want = std::max(1, kPlanBlocks / a.g.n_kv - y.sets);
    // each set's last split may be short
    y.works = y.want ? std::min<long long>(y.want + y.sets, y.sets * std::min<long long>(kMaxSplits, units)) : y.sets;
    return y;
}

}  // namespace

size_t attention_paged_workspace_bytes(const PagedAttnArgs& a)
{
    const Layout y = layout_of(a);
    return y.want ? attention_counter_bytes() + (size_t)y.works * a.g.n_kv * y.cols * (a.head_dim + 2) * sizeof(float) : 0;
}

hipError_t launch_attention_paged(const PagedAttnArgs& a, float* workspace, hipStream_t st)
{
    const Layout y = layout_of(a);
    MmaArgs A{};
    A.a = a;
    A.group = y.group;
    A.cols = y.cols;
    A.tiles = y.tiles;
    A.sets = y.sets;
    A.want = y.want;
    A.cap = a.g.max_blocks * a.g.tpb;
    A.tpb_shift = (a.g.tpb & (a.g.tpb - 1)) == 0 ? __builtin_ctz((unsigned)a.g.tpb) : -1;
    A.counters = reinterpret_cast<uint32_t*>(workspace);
    A.part = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + attention_counter_bytes());
    A.part_bytes = (uint32_t)((size_t)y.works * a.g.n_kv * y.cols * (a.head_dim + 2) * sizeof(float));  // below 2^31: plan()'s blocks
    const unsigned rows_of_grid = (unsigned)std::min<long long>(y.works, 32768);
    const dim3 grid((unsigned)a.g.n_kv, rows_of_grid, (unsigned)((y.works + rows_of_grid - 1) / rows_of_grid));
    by_shape(a.ks != nullptr, a.head_dim, [&](auto q, auto hd) {
        constexpr bool Q8 = decltype(q)::value;
        constexpr int HD = decltype(hd)::value;
        const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, st, A); };
        if constexpr (HD <= 128) {
            if (y.ct == 2) return a.cap > 0.0f ? go(attn_paged_kernel<Q8, HD, 2, true>) : go(attn_paged_kernel<Q8, HD, 2, false>);
        }
        a.cap > 0.0f ? go(attn_paged_kernel<Q8, HD, 1, true>) : go(attn_paged_kernel<Q8, HD, 1, false>);
    });
    return hipGetLastError();
}

}  // namespace cellm
