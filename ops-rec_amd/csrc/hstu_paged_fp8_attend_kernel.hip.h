// HSTU attention over the 8-bit paged cache (gfx950).
//
//   S = Q K^T,  P = silu(alpha S) * silu_scale * M,  O = P V,  with K and V the codes of the cache times their blocks' scales
//
// A step is one block of 32 keys, which lies in one page and has one scale for K and one for V.  Both products run on
// v_mfma_f32_32x32x16 in the type of q, which holds an e4m3 value exactly; bf16 also holds it times the scale, a power of two (below
// 2^-126 not all of its bits), which v_cvt_scalef32_pk multiplies by while it converts, so that scales cost nothing.  fp16 does not: see Fp8Unit.
//   S^T[key][row] = K . Q^T     A = K: lane l % 32 takes key pi(l % 32) of the block, 16 dims of its half at a time; B = Q, in
//                               registers from the start, the same dims
//   O^T[dim][row] += V^T . P^T  A = V^T: lane l % 32 takes dim pi(l % 32) of a group of 32, the 16 keys of its half; B = P
// The rows of the 32x32 result that a lane holds are 8 a + 4 half + b (a, b = 0 .. 3).  With pi(8 a + 4 h + b) = 16 h + 4 a + b a
// lane's 16 values of S are the keys 16 half .. + 15 in order, which is what the second product wants of B when A's lanes load 16
// consecutive keys: P goes from one product to the other in its registers, V (stored with the keys innermost) comes straight from
// memory, and no value passes through LDS or another lane.  The same order of V's dims gives a lane 16 consecutive output dims.
//
// The columns of the result are rows of q: (row, query head of the key head's group) pairs, head fastest, so that grouped heads
// share the keys that are read.
//
// A workgroup's wavefronts take the blocks of its 32 columns in turn, each converting what it reads, one block ahead in registers, and add
// their outputs through LDS at the end: no barrier until then.  Bound by the bytes of the codes where columns are few (64 x 4 key heads of
// one row on 2048 .. 8192 keys, d 128, 339 MB in 75 us, 4.5 TB/s; 3 x 2 of 30011 .. 120011, d 256, 231 MB in 51), else by a wavefront's chain
// from load to product (about 1 us a step, 4 us before the first: 32 x 4 of 49 .. 64 rows on 501 .. 4001, d 64, 24 us).
#pragma once
#include "hstu_paged_fp8_common.hip.h"
#include "hstu_paged_fp8_variants.h"

namespace hstu {

typedef __attribute__((ext_vector_type(4))) float f32x4_t;

// One 16-byte chunk of codes as eight + eight 16-bit values.
struct Fp8Pair {
    u32x4_t lo, hi;
};
template <typename Tag>
__device__ __forceinline__ uint32_t fp8_two(uint32_t codes, float scale, bool hi);
template <>
__device__ __forceinline__ uint32_t fp8_two<bf16_tag>(uint32_t codes, float scale, bool hi)
{
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
}
template <>
__device__ __forceinline__ uint32_t fp8_two<f16_tag>(uint32_t codes, float scale, bool hi)
{
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
}
template <typename Tag>
__device__ __forceinline__ Fp8Pair fp8_widen(u32x4_t codes, float scale)
{
    Fp8Pair r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        r.lo[2 * i] = fp8_two<Tag>(codes[i], scale, false);
        r.lo[2 * i + 1] = fp8_two<Tag>(codes[i], scale, true);
        r.hi[2 * i] = fp8_two<Tag>(codes[2 + i], scale, false);
        r.hi[2 * i + 1] = fp8_two<Tag>(codes[2 + i], scale, true);
    }
    return r;
}

// A cache has no type, and fp16 does not hold what a code times its scale may be (from 65520 on it would be infinite, and zero times that
// NaN in rows that do not see the key; below 2^-14 it would be rounded), nor what a weight may be before alpha and silu_scale. So for
// rows of fp16 the products run on the codes themselves, which fp16 holds exactly. A block's scale of K goes into the exponent of silu,
// and the weights go into the second product times both scales, in units of their row's own. Of a row of dim values up to m a score in
// units of K's scale is at most 448 dim m; the unit is a power of two that puts this bound, times the scales of a block that the row has
// seen a key of, below 2^11, and is changed, the row's sums with it, by a block whose scales' product is 2^5 times that block's or more,
// or less than 2^-8 of it. Weights are then rounded to multiples of 2^-24 of a unit at worst, 2^-25 of what the bound says for their
// block; a score's own sum in fp32 is good to 2^-24 of it. (A row is a column of the result: a lane holds of its own row only, and so
// does the lane of the same row in the other half. Nothing that a row does not see changes its unit, and a block that holds one value of
// 1e30 leaves the sums of other blocks as they are.) It costs no instruction an element: x / (1 + e) * 2^n is x / (e 2^-n + 2^-n). bf16
// reaches as far as fp32 and needs none of this.
struct Fp8Unit {
    int own;      // exponent of the unit's reciprocal for a block with scales of 1
    int up;       // and as it is: the unit is 2^-up; ahead of the first block one that none fits
    bool finite;  // the row
    static __device__ __forceinline__ int exponent(float power_of_two)
    {
        return static_cast<int>(__builtin_bit_cast(uint32_t, power_of_two) >> 23 & 0xffu) - 127;
    }
    // what `x` is in the two lanes of this lane's row, the larger of them
    static __device__ __forceinline__ uint32_t of_row(uint32_t x)
    {
        const u32x2_t two = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        const uint32_t lower = two[0], upper = two[1];
        return lower > upper ? lower : upper;
    }
    template <int NC>
    __device__ __forceinline__ Fp8Unit(const u32x4_t (&q)[NC][2], int dim)
    {
        typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
        u16x2_t top = {0, 0};
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t word = q[n][i >> 2][i & 3];
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, word & 0x7fff7fffu));
            }
        }
        const uint32_t a = top[0], b = top[1], m = of_row(a > b ? a : b);
        finite = m < 0x7c00u;
        const int bits = 32 - __builtin_clz(static_cast<uint32_t>(dim) - 1);  // dim <= 2^bits, codes <= 2^9
        own = 11 - (__builtin_amdgcn_frexp_expf(lo_to_float<f16_tag>(m)) + 9 + bits);
        up = own + 1024;
    }
    // Makes the unit fit a block whose scales' exponents add up to `by`, of which this row sees keys (`sees`, the same in both lanes of
    // a row).
    template <int NC>
    __device__ __forceinline__ void fit(f32x16_t (&acc)[NC], int by, bool sees)
    {
        const bool other = sees & (static_cast<uint32_t>(up + by - own + 8) > 12u);
        if (__any(other)) {
            // (the sums stay below 2^100, of which a smaller unit for a block of far smaller scales would leave nothing finite)
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = acc[n][i];
                    sum = __builtin_fmaxf(sum, __builtin_fabsf(x));
                }
            }
            sum = __builtin_bit_cast(float, of_row(__builtin_bit_cast(uint32_t, sum)));
            const int left = 100 - __builtin_amdgcn_frexp_expf(sum), room = sum > 0.0f ? (left > 0 ? left : 0) : 4096;
            const int wanted = own - by - up, change = other ? (wanted < room ? wanted : room) : 0;
            up += change;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    acc[n][i] = __builtin_ldexpf(acc[n][i], change);
                }
            }
        }
    }
    // What the denominators of a block's weights are multiplied by.  (One over it is at most 2^25 for a row that sees a key of the block, others have
    // scores of zero; and of scores, below 2^33, 2^-64 leaves nothing in fp16.)
    __device__ __forceinline__ float denominator(int by) const
    {
        const int n = up + by;
        return __builtin_ldexpf(1.0f, -(n > 64 ? 64 : (n < -64 ? -64 : n)));
    }
    // what a weight in units is multiplied by, without the scale of V of exponent `v`
    __device__ __forceinline__ float weight(int v) const { return __builtin_ldexpf(1.0f, -up - v); }
    template <int NC>
    __device__ __forceinline__ void undo(f32x16_t (&acc)[NC]) const
    {
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                acc[n][i] = __builtin_ldexpf(acc[n][i], -up);
            }
        }
    }
};
// whether some of a lane's 16 scores, or of the other's of its row, is not zero
__device__ __forceinline__ bool fp8_some_score(const float (&x)[16])
{
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float one = x[i];
        bits |= __builtin_bit_cast(uint32_t, one);
    }
    return Fp8Unit::of_row(bits & 0x7fffffffu) != 0;
}
// silu of 16 scores x (in units of a scale 2^k) without alpha, in units of a row: x / (1 + 2^(c_exp 2^k x)) times 1 / g.  `most`: of k, that leaves
// the product finite (a score of 0 has a weight of 0).
__device__ __forceinline__ void fp8_weights_in_units(float (&x)[16], float c_exp, int k, int most, float g)
{
    const float c = __builtin_ldexpf(c_exp, k < most ? k : most);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        x[i] = x[i] * __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_amdgcn_exp2f(x[i] * c), g, g));
    }
}
__device__ __forceinline__ int fp8_most_scale(float c_exp) { return uniform(127 - __builtin_amdgcn_frexp_expf(c_exp)); }

// 0x80 in the place of each of four codes that is NaN (0x7f, 0xff), 0 elsewhere
__device__ __forceinline__ uint32_t nan_codes(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ u32x4_t load_codes(__amdgpu_buffer_rsrc_t rsrc, uint32_t offset)
{
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(offset), 0, 0));
}

// The blocks that some row of a range of rows sees, in at most three runs: the first tokens (sinks), what the window or the
// whole history leaves up to the targets, and the targets' own groups.
struct Fp8Runs {
    int n_a, n_b, n_c;  // blocks of each
    int b0, c0;         // first block of the second and of the third
    __device__ __forceinline__ int count() const { return n_a + n_b + n_c; }
    __device__ __forceinline__ int block(int n) const { return n < n_a ? n : (n < n_a + n_b ? b0 + n - n_a : c0 + n - n_a - n_b); }
};

// What a sequence's rows see: row i (position p = i + len - rows) sees the keys j <= p; a target row, of the last `targets`, not
// the targets of the groups above its own; with a window only j > centre - window and j < sinks, the centre being p, or for a
// target row the first target.
struct Fp8Mask {
    int len, delta, first_target, first_key, group, window, sinks;
    bool targets;

    __device__ __forceinline__ int lim(int i) const  // one past the last key
    {
        const int e = i + delta + 1;
        return e < 0 ? 0 : (e > len ? len : e);
    }
    __device__ __forceinline__ int hole(int i) const  // keys [first_key, hole) are not seen
    {
        return targets && i >= first_target ? first_key + (i - first_target) / group * group : first_key;
    }
    __device__ __forceinline__ int low(int i) const  // keys [sinks, low) are not seen
    {
        const int centre = targets && i >= first_target ? first_key : i + delta;
        return window > 0 ? centre - window + 1 : 0;
    }
};

__device__ __forceinline__ Fp8Runs fp8_runs(const Fp8Mask& m, int i0, int i1)  // rows [i0, i1), i0 < i1
{
    Fp8Runs r;
    const int end = (m.lim(i1 - 1) + kFp8Block - 1) / kFp8Block;
    const int low = m.low(i0) > 0 ? m.low(i0) / kFp8Block : 0;
    const int sinks = m.window > 0 && m.sinks > 0 ? (m.sinks + kFp8Block - 1) / kFp8Block : 0;
    r.n_a = sinks < low ? (sinks < end ? sinks : end) : 0;
    const int b = sinks < low ? low : 0;  // (0: the window reaches the first tokens, one run)
    r.b0 = b;
    // the blocks that lie whole in what even the first row does not see of the targets
    int h0 = end, h1 = end;
    const int hole = m.hole(i0);
    if (hole > m.first_key && m.first_key >= 0) {
        h0 = (m.first_key + kFp8Block - 1) / kFp8Block;
        h1 = hole / kFp8Block;
        if (h1 <= h0 || h0 < b) {
            h0 = h1 = end;
        }
    }
    h0 = h0 < end ? h0 : end;
    h1 = h1 < end ? h1 : end;
    r.n_b = h0 > b ? h0 - b : 0;
    r.c0 = h1;
    r.n_c = end > h1 ? end - h1 : 0;
    return r;
}

// The blocks that every row of [i0, i1] sees whole: an interval, and the first few of the sinks.
struct Fp8Whole {
    int lo, hi, sinks;
    __device__ __forceinline__ bool has(int blk) const { return static_cast<uint32_t>(blk - lo) < static_cast<uint32_t>(hi - lo) || blk < sinks; }
};
__device__ __forceinline__ Fp8Whole fp8_whole(const Fp8Mask& m, int i0, int i1)
{
    Fp8Whole w;
    const int lim = m.lim(i0), low = m.low(i1);
    const int end = m.hole(i1) > m.first_key ? (lim < m.first_key ? lim : m.first_key) : lim;  // (up to the targets where some are not seen)
    w.lo = uniform(low > 0 ? (low + kFp8Block - 1) / kFp8Block : 0);
    w.hi = uniform(end > 0 ? end / kFp8Block : 0);
    w.hi = w.hi < w.lo ? w.lo : w.hi;
    const int sinks = m.window > 0 ? (m.sinks < end ? m.sinks : end) : 0;
    w.sinks = uniform(sinks > 0 ? sinks / kFp8Block : 0);
    return w;
}

// One sequence of a call: its rows of q, its pages and live keys, and what its rows see.
struct Fp8Item {
    Fp8Sequence seq;
    int64_t q0, q1;  // rows of q
    int n_rows;      // of them within the longest length allowed
    Fp8Mask mask;
};
__device__ __forceinline__ Fp8Item fp8_item(const Fp8AttendArgs& a, int b)
{
    const Fp8Cache& c = a.c;
    Fp8Item it;
    it.seq = fp8_sequence(c, b);
    it.seq.len = it.seq.len < a.max_k ? it.seq.len : a.max_k;
    int64_t q0 = load_index_uniform(a.offs_q, b, c.idx64), q1 = load_index_uniform(a.offs_q, b + 1, c.idx64);
    q0 = q0 < 0 ? 0 : (q0 > a.total_q ? a.total_q : q0);
    q1 = q1 < q0 ? q0 : (q1 > a.total_q ? a.total_q : q1);
    it.q0 = q0;
    it.q1 = q1;
    it.n_rows = static_cast<int>(q1 - q0 < a.max_q ? q1 - q0 : a.max_q);
    int n_targets = 0;
    if (a.num_target != nullptr && a.group > 0) {
        const int64_t t = load_index_uniform(a.num_target, b, c.idx64);
        n_targets = static_cast<int>(t < 0 ? 0 : (t > 0x3fffffff ? 0x3fffffff : t));
    }
    Fp8Mask& m = it.mask;
    m.len = it.seq.len;
    m.delta = it.seq.len - it.n_rows;
    m.targets = n_targets > 0;
    m.first_target = it.n_rows - n_targets;
    m.first_key = it.seq.len - n_targets;
    m.group = m.targets ? a.group : 1;
    m.window = a.window;
    m.sinks = a.sinks;
    return it;
}

// Which share of a sequence's keys a workgroup takes.  Tiles whose keys take long are dealt to several workgroups, in parts of as
// many blocks each, `chunk`, whatever the sequence: with up to 64 sequences, a lane of a wavefront for each, the lengths are
// looked at, and the chunk is what makes hardly fewer than total_parts of them all -- sum ceil(blocks / chunk) is at most sum blocks / chunk +
// the number of sequences, and about half that number less on average (16 x 4 pairs of 1024 rows on 2048 .. 8192 keys 259 us by the bound,
// 248 by the half).  (Cut alike by the longest length allowed, parts of short sequences have nothing to do: 3 x 2 key heads
// of 30011 .. 120011 keys, d 256, 70 us in such parts, 48 in these.)  First come the first parts of all sequences, the longest first,
// then their second parts, and so on: what starts late is short.
struct Fp8Deal {
    int b;      // the sequence; -1: none
    int part;   // of its
    int parts;
    int chunk;
    int slot;   // number of the part among all, in the order of the sequences (of a sequence that has one: unused)
};
struct Fp8DealLanes {
    int chunk, parts, rank;  // of the sequence of this lane: its parts (0: no sequence), and how many come before it
    // number of the first of the p-th parts of all
    __device__ __forceinline__ int count(int p) const { return static_cast<int>(__popcll(__ballot(parts > p))); }
};
__device__ __forceinline__ Fp8DealLanes fp8_deal_lanes(const Fp8AttendArgs& a)
{
    const int lane = threadIdx.x & 63, n = a.c.n_batch;
    const int64_t len = load_index(a.c.cache_len, lane < n ? lane : 0, a.c.idx64);
    const int keys = static_cast<int>(len < 0 ? 0 : (len < a.max_k ? len : a.max_k));
    const int all = (keys + kFp8Block - 1) / kFp8Block, blocks = lane < n ? (all < a.most_blocks ? all : a.most_blocks) : -1;
    const auto over_lanes = [](int x) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            x += __shfl_xor(x, d, 64);
        }
        return uniform(x);
    };
    const int mine = blocks > 0 ? blocks : 0, sum = over_lanes(mine);
    Fp8DealLanes r;
    // the first that makes no more than total_parts: sequences' last parts taken to be a half, or a quarter of a part on average, or nothing
#pragma unroll
    for (int lost = 2; lost <= 4; ++lost) {
        const int whole = a.total_parts - div_small(lost * n, 4), even = uniform((sum + whole - 1) / whole);
        r.chunk = even > a.chunk ? even : a.chunk;
        const int parts = div_small(mine + r.chunk - 1, r.chunk);
        r.parts = lane < n ? (parts > 1 ? parts : 1) : 0;
        if (lost == 4 || over_lanes(r.parts) <= a.total_parts) {
            break;
        }
    }
    r.rank = 0;
    for (int l = 0; l < n; ++l) {
        const int other = __builtin_amdgcn_readlane(blocks, l);
        r.rank += (other > blocks) | ((other == blocks) & (l < lane)) ? 1 : 0;
    }
    return r;
}
__device__ __forceinline__ Fp8Deal fp8_deal(const Fp8AttendArgs& a, int n)  // the n-th part of all
{
    if (a.total_parts == 0) {
        return {n < a.c.n_batch ? n : -1, 0, 1, 0x3fffffff, n};
    }
    if (a.c.n_batch > 64) {
        const int b = uniform(n / a.parts);
        return {b < a.c.n_batch ? b : -1, n - b * a.parts, a.parts, a.chunk, n};
    }
    const Fp8DealLanes l = fp8_deal_lanes(a);
    int part = 0, rank = n, count = l.count(0);
    while (rank >= count && count > 0) {
        rank -= count;
        count = l.count(++part);
    }
    const uint64_t mine = __ballot((l.rank == rank) & (l.parts > part));
    const int b = mine != 0 ? __builtin_ctzll(mine) : -1;
    const int parts = mine != 0 ? __builtin_amdgcn_readlane(l.parts, b >= 0 ? b : 0) : 1;
    int ahead = 0;  // parts of the sequences before
    if (parts > 1) {
        ahead = static_cast<int>(threadIdx.x & 63) < b ? l.parts : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            ahead += __shfl_xor(ahead, d, 64);
        }
    }
    return {b, part, parts, l.chunk, uniform(ahead) + part};
}

// What a workgroup does: slots are (part, key head) x row tile of the launch, the tiles of a part and head, which read the same keys, on one XCD
// (workgroup w runs on XCD w mod 8).
__device__ __forceinline__ Fp8Deal fp8_slot(const Fp8AttendArgs& a, int& g, int& tile)
{
    const int slot = static_cast<int>(blockIdx.x);
    int unit = slot;
    tile = 0;
    if (a.row_tiles > 1) {
        const int oct = uniform(slot / (8 * a.row_tiles)), rest = slot - oct * 8 * a.row_tiles;
        unit = oct * 8 + (rest & 7);
        tile = a.row_tiles - 1 - (rest >> 3);  // (later rows see more keys: first)
    }
    const int n = uniform(unit / a.c.n_heads);
    g = unit - n * a.c.n_heads;
    return fp8_deal(a, n);
}

// Rows of no sequence, and rows past the longest sequence allowed: zeros.  For the workgroup of a pair's first tile and part.
template <int THREADS>
__device__ __forceinline__ void fp8_clear_rows(const Fp8AttendArgs& a, const Fp8Item& item, int b, int g, uint16_t* out)
{
    const int64_t pitch = static_cast<int64_t>(a.n_heads_q) * a.c.dim, mine = static_cast<int64_t>(a.ratio) * a.c.dim;
    const auto clear = [&](int64_t from, int64_t to) {
        for (int64_t r = from; r < to; ++r) {
            for (int64_t x = threadIdx.x; x < mine; x += THREADS) {
                out[r * pitch + g * mine + x] = 0;
            }
        }
    };
    clear(item.q0 + item.n_rows, item.q1);
    if (b == 0) {
        clear(0, item.q0);
    }
    if (b == a.c.n_batch - 1) {
        clear(item.q1, a.total_q);
    }
}

// x of another lane of its row of 16, as a DPP control says
template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// halves the N values a lane carries: a lane with `upper` keeps the second half, and every lane adds what its partner gives away
template <int CTRL, int N>
__device__ __forceinline__ void halve(float (&v)[16], bool upper)
{
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float give = upper ? v[i] : v[i + N / 2], keep = upper ? v[i + N / 2] : v[i];
        v[i] = keep + dpp<CTRL>(give);
    }
}
// The sums of 16 values over the 32 lanes of each half, in the vector unit alone (through LDS the exchanges took longer than the block's
// products).  Returned to lanes 2 x and 2 x + 1 is that of the key whose bits are those of x, highest first.
__device__ __forceinline__ float fp8_key_sum(float (&v)[16], int lane)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // rows of 16 lanes, in pairs: the odd row of one against the even row of the other
        const u32x2_t r =
            __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v[i]), __builtin_bit_cast(uint32_t, v[i + 8]), false, false);
        const uint32_t one = r[0], other = r[1];  // (values: a bit cast of an element of a vector takes its first)
        v[i] = __builtin_bit_cast(float, one) + __builtin_bit_cast(float, other);
    }
    halve<0x128, 8>(v, (lane & 8) != 0);  // row_ror:8
    halve<0x141, 4>(v, (lane & 4) != 0);  // row_half_mirror: 7 - l of each eight
    halve<0x4e, 2>(v, (lane & 2) != 0);   // quad_perm 2 3 0 1
    return v[0] + dpp<0xb1>(v[0]);        // quad_perm 1 0 3 2
}
__device__ __forceinline__ void fp8_store_key_sum(const Fp8AttendArgs& a, float sum, int lane, int pair, int row_tile, int row_tiles, int blk, int lin)
{
    if ((lane & 1) == 0) {
        const int key = 16 * (lane >> 5) + 8 * ((lane >> 4) & 1) + 4 * ((lane >> 3) & 1) + 2 * ((lane >> 2) & 1) + ((lane >> 1) & 1);
        if (a.weight_partial != nullptr) {
            a.weight_partial[((static_cast<int64_t>(pair) * row_tiles + row_tile) * a.max_blocks + blk) * kFp8Block + key] = sum;
        } else if (lin >= 0) {  // (a page may be in two sequences)
            unsafeAtomicAdd(a.c.weights + static_cast<int64_t>(lin) * kFp8Block + key, sum);
        }
    }
}

constexpr uint32_t kV32 = 32 * kFp8Block;  // bytes of 32 dims of V of a block

// Outputs that a value which is NaN reaches, of one block: a product of ones at the codes for NaN with the 0 / 1 mask counts, for every
// (dim, row), the NaN that the row sees.  j0: the first key of this lane's half; v_at: where its codes of the first 32 dims are.  (The products proper
// had zeros in the place of those codes.)
template <typename Tag, int NC, typename Sees>
__device__ __forceinline__ void fp8_poison(f32x16_t (&acc)[NC], const Fp8Cache& c, int lin, uint32_t v_at, int j0, int len, Sees sees)
{
    const uint32_t bytes = static_cast<uint32_t>(kFp8Block) * c.dim;
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(c.v + static_cast<int64_t>(lin < 0 ? 0 : lin) * bytes, lin < 0 ? 0u : bytes);
    u32x4_t seen[2];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const int j = j0 + i;
        seen[i >> 3][(i >> 1) & 3] = pack2<Tag>(((j < len) & sees(j)) ? 1.0f : 0.0f, ((j + 1 < len) & sees(j + 1)) ? 1.0f : 0.0f);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        u32x4_t ones = load_codes(rsrc, v_at + n * kV32);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ones[i] = (nan_codes(ones[i]) >> 7) * 0x38u;  // the code of 1
        }
        const Fp8Pair oo = fp8_widen<Tag>(ones, 1.0f);
        f32x16_t hits = mfma32<Tag>(oo.lo, seen[0], f32x16_t{0.0f});
        hits = mfma32<Tag>(oo.hi, seen[1], hits);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[n][i] = hits[i] > 0.0f ? __builtin_nanf("") : acc[n][i];
        }
        __builtin_amdgcn_sched_barrier(0);  // (a group of dims at a time: no registers are set aside for this)
    }
}

// that a variant's registers allow without scratch
constexpr int fp8_wavefronts_per_simd(int nc, bool weights) { return nc <= 2 ? (nc == 2 && weights ? 3 : 4) : (nc <= 4 ? 2 : 1); }

// Tag     : type of q and out
// NC      : groups of 32 dims (dim is at most 32 NC, a multiple of 16)
// WK      : wavefronts of a workgroup, over the keys of a tile of rows
// WEIGHTS : the sums of |P| per key as well
template <typename Tag, int NC, int WK, bool WEIGHTS>
__global__ __launch_bounds__(64 * WK) __attribute__((amdgpu_waves_per_eu(fp8_wavefronts_per_simd(NC, WEIGHTS)))) void hstu_paged_fp8_attend_kernel(const Fp8AttendArgs a)
{
    constexpr int T = 64 * WK, TILE = kFp8KeysRows;
    constexpr bool F16 = __is_same(Tag, f16_tag);
    constexpr int CHUNK_WORDS = 64 * 16;
    __shared__ __attribute__((aligned(16))) float s_sum[2][WK * CHUNK_WORDS];

    const Fp8Cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wk = uniform(tid >> 6);
    const int col = lane & 31, half = lane >> 5;

    int g, tile;
    const Fp8Deal deal = fp8_slot(a, g, tile);
    if (deal.b < 0) {
        return;
    }
    const int b = deal.b, part = deal.part, pair = b * c.n_heads + g;

    const Fp8Item item = fp8_item(a, b);
    const Fp8Sequence& seq = item.seq;
    const Fp8Mask& mask = item.mask;
    const int64_t q0 = item.q0, q1 = item.q1;
    const int n_rows = item.n_rows;
    const int dim = c.dim;
    uint16_t* const out = static_cast<uint16_t*>(a.out);

    if (a.tile_first + tile == 0 && part == 0) {
        fp8_clear_rows<T>(a, item, b, g, out);
    }
    const int n_pairs_rows = n_rows * a.ratio;  // (row, head) pairs
    const int m0 = (a.tile_first + tile) * TILE, m1 = m0 + TILE < n_pairs_rows ? m0 + TILE : n_pairs_rows;
    if (m0 >= m1) {
        return;
    }
    // what the workgroup sweeps: the blocks of its tile's rows
    const int i_first = uniform(div_small(m0, a.ratio)), i_last = uniform(div_small(m1 - 1, a.ratio));
    Fp8Runs runs = fp8_runs(mask, i_first, i_last + 1);
    runs = {uniform(runs.n_a), uniform(runs.n_b), uniform(runs.n_c), uniform(runs.b0), uniform(runs.c0)};
    const int n_blocks = runs.count();
    const int parts_used = deal.parts == 1 ? 1 : uniform((n_blocks + deal.chunk - 1) / deal.chunk);
    if (part > 0 && part >= parts_used) {
        return;
    }
    if (part == 0 && a.joins != nullptr && threadIdx.x == 0) {
        a.joins[pair * a.row_tiles + tile] = int2{parts_used < deal.parts ? parts_used : deal.parts, deal.slot};
    }
    const int n_begin = deal.parts == 1 ? 0 : part * deal.chunk;
    const int n_end = part == deal.parts - 1 || n_blocks - n_begin < deal.chunk ? n_blocks : n_begin + deal.chunk;

    // q: the rows of this wavefront, 16 dims of this lane's half per group of 32
    u32x4_t q[NC][2];
    const int m = m0 + col, i_row = div_small(m < n_pairs_rows ? m : 0, a.ratio);
    const int lim = m < n_pairs_rows ? mask.lim(i_row) : 0, hole = mask.hole(i_row), low = mask.low(i_row);
    {
        const uint32_t bytes = static_cast<uint32_t>(n_rows) * static_cast<uint32_t>(a.n_heads_q) * dim * 2u;
        const __amdgpu_buffer_rsrc_t rsrc =
            make_rsrc(static_cast<const uint16_t*>(a.q) + q0 * a.n_heads_q * static_cast<int64_t>(dim), bytes);
        const uint32_t at = (static_cast<uint32_t>(i_row) * a.n_heads_q + g * a.ratio + (m - i_row * a.ratio)) * dim * 2u;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 32 * n + 16 * half + 8 * u;
                q[n][u] = load_codes(rsrc, m < n_pairs_rows && d < dim ? at + d * 2u : kOutOfRange);
            }
        }
    }

    // offsets of this lane's chunks within a block of codes; dims past the last read as zeros
    const int pi = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
    const uint32_t block_bytes = static_cast<uint32_t>(kFp8Block) * dim;
    uint32_t k_at[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int d = 32 * n + 16 * half;
        k_at[n] = d < dim ? static_cast<uint32_t>(pi) * dim + d : kOutOfRange;
    }
    const uint32_t v_at = static_cast<uint32_t>(pi) * kFp8Block + 16 * half;  // (32 dims on: kV32 on; V of a dim past the last lies past the block)

    f32x16_t acc[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        acc[n] = f32x16_t{0.0f};
    }

    const Fp8Whole whole_blocks = fp8_whole(mask, i_first, i_last);  // these need no mask

    // Steps of this wavefront: blocks n_begin + wk, + WK, ...; the places and scales of 64 of them at a time, a step per lane.  They are
    // looked up, and handed out by readlane, with every lane active: a lane that is not has no value that another may count on (the
    // compiler may move a value between registers under the mask of a branch).
    const int n_steps = n_end - n_begin - wk > 0 ? (n_end - n_begin - wk + WK - 1) / WK : 0;
    int my_lin = -1;
    float my_ks = 1.0f, my_vs = 1.0f;
    const auto look_up = [&](int base) {  // (base < n_steps; lanes behind the last step take it too)
        const int s = base + lane < n_steps ? base + lane : n_steps - 1;
        my_lin = fp8_block(c, c.page_ids, seq.first, g, runs.block(n_begin + wk + s * WK));
        const int at = my_lin >= 0 ? my_lin : 0;
        const float ks = c.k_scale[at], vs = c.v_scale[at];
        my_ks = my_lin >= 0 ? ks : 1.0f;  // (a page that is none holds zeros, and zero times what another block has may not be that)
        my_vs = my_lin >= 0 ? vs : 1.0f;
    };
    const auto place_of = [&](int s) { return __builtin_amdgcn_readlane(my_lin, s & 63); };

    struct Stage {
        u32x4_t k[NC], v[NC];
    };
    const auto request = [&](Stage& st, int s) {
        const int lin = place_of(s);
        const int64_t at = static_cast<int64_t>(lin < 0 ? 0 : lin) * block_bytes;
        const __amdgpu_buffer_rsrc_t kr = make_rsrc(c.k + at, lin < 0 ? 0u : block_bytes), vr = make_rsrc(c.v + at, lin < 0 ? 0u : block_bytes);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            st.k[n] = load_codes(kr, k_at[n]);
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            st.v[n] = load_codes(vr, v_at + n * kV32);
        }
    };
    const auto sees_key = [&](int j) {  // whether this lane's row sees key j
        return static_cast<bool>((j < lim) & ((j < mask.first_key) | (j >= hole)) & ((j >= low) | (j < mask.sinks)));
    };
    bool poisoned = false;
    Fp8Unit unit(q, dim);  // (fp16)
    const int most_scale = fp8_most_scale(a.c_exp);
    const auto step = [&](Stage& st, int s, float ks, float vs) {
        const int lin = place_of(s);
        const int blk = runs.block(n_begin + wk + s * WK), c0 = blk * kFp8Block;
        const bool whole = whole_blocks.has(blk);
        const int by = Fp8Unit::exponent(ks) + Fp8Unit::exponent(vs);
        if (F16 && whole) {
            unit.fit<NC>(acc, by, true);
        }
        f32x16_t sc = f32x16_t{0.0f};
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const Fp8Pair kk = fp8_widen<Tag>(st.k[n], F16 ? 1.0f : ks);
            sc = mfma32<Tag>(kk.lo, q[n][0], sc);
            sc = mfma32<Tag>(kk.hi, q[n][1], sc);
        }
        const int end = c0 + kFp8Block;
        // P goes into the second product rounded to the type of q.  What that leaves of half the keys (0 .. 7 and 16 .. 23 of a block) goes into a
        // product of its own, so that P adds less to the error than the output's rounding: bf16 outputs of few rows would else be 1.4 to
        // 1.5 times as far off as rounding them alone, and are 1.2 times.  (64 rows of one query 74 us without and 75 with it, 32 x 4 pairs of 49 .. 64
        // rows 20 and 22; the other half as well would be 2 more.)
        u32x4_t p[2], rest;
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = sc[i];
            w[i] = F16 ? x : x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * a.c_exp));
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = sees_key(c0 + 16 * half + i) ? w[i] : 0.0f;
            }
            if constexpr (F16) {
                unit.fit<NC>(acc, by, fp8_some_score(w));
            }
        }
        if constexpr (F16) {
            fp8_weights_in_units(w, a.c_exp, Fp8Unit::exponent(ks), most_scale, unit.denominator(by));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w0 = w[8 * u + 2 * i], w1 = w[8 * u + 2 * i + 1];
                const uint32_t two = pack2<Tag>(w0, w1);
                p[u][i] = two;
                if (u == 0) {
                    rest[i] = pack2<Tag>(w0 - lo_to_float<Tag>(two), w1 - hi_to_float<Tag>(two));
                }
            }
        }
        bool beyond = !unit.finite;  // what is infinite in the type of q leaves nothing, not NaN
        if constexpr (!F16) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                top = __builtin_fmaxf(top, __builtin_fabsf(w[i]));
            }
            beyond = top > 3.3895314e38f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            rest[i] = beyond ? 0u : rest[i];
        }
        if (end > seq.len) {  // codes behind the last row may be anything, NaN among them: zero times that is not zero
            const int left = seq.len - c0 - 16 * half;  // live keys of this lane's sixteen
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = left - 4 * i;
                const uint32_t keep = n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    st.v[k][i] &= keep;
                }
            }
        }
        // A key that some rows do not see must not reach them, and zero times NaN would.  The codes for NaN are found by their bits; where
        // a block with a mask holds one, the products run on zeros in their place, and what they make NaN is seen to after the sweep.
        if (!whole) {
            uint32_t any = 0;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bits = nan_codes(st.v[n][i]);
                    any |= bits;
                    st.v[n][i] &= ~((bits >> 7) * 0xffu);
                }
            }
            poisoned = poisoned || __any(any != 0);
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const Fp8Pair vv = fp8_widen<Tag>(st.v[n], F16 ? 1.0f : vs);
            acc[n] = mfma32<Tag>(vv.lo, p[0], acc[n]);
            acc[n] = mfma32<Tag>(vv.hi, p[1], acc[n]);
            acc[n] = mfma32<Tag>(vv.lo, rest, acc[n]);
        }
        if constexpr (WEIGHTS) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = F16 ? __builtin_fabsf(w[i]) * unit.weight(Fp8Unit::exponent(vs)) : __builtin_fabsf(w[i]);
            }
            const float all = fp8_key_sum(w, lane) * __builtin_fabsf(a.c_out);
            fp8_store_key_sum(a, all, lane, pair, tile, a.row_tiles, blk, lin);
        }
    };
    const auto scale_of = [&](float mine, int s) {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), s & 63));
    };

    Stage st[2];
    for (int base = 0; base < n_steps; base += 64) {
        look_up(base);
        const int stop = n_steps < base + 64 ? n_steps : base + 64;
        request(st[0], base);
        for (int s = base; s < stop; s += 2) {
            if (s + 1 < stop) {
                request(st[1], s + 1);
            }
            step(st[0], s, scale_of(my_ks, s), scale_of(my_vs, s));
            if (s + 1 < stop) {
                if (s + 2 < stop) {
                    request(st[0], s + 2);
                }
                step(st[1], s + 1, scale_of(my_ks, s + 1), scale_of(my_vs, s + 1));
            }
        }
    }

    if (poisoned) {
        for (int s = 0; s < n_steps; ++s) {
            const int blk = runs.block(n_begin + wk + s * WK);
            if (whole_blocks.has(blk)) {
                continue;
            }
            const int lin = uniform(fp8_block(c, c.page_ids, seq.first, g, blk));
            fp8_poison<Tag, NC>(acc, c, lin, v_at, blk * kFp8Block + 16 * half, seq.len, sees_key);
        }
    }

    if constexpr (F16) {
        unit.undo<NC>(acc);
    }
    // ---- the sum over the wavefronts that shared the keys, and the store ----
    const int lane_e = lane_here(), tid_e = 64 * wk + lane_e, half_e = lane_e >> 5, ratio = here(a.ratio);
    const bool partial = parts_used > 1 && deal.parts > 1;
    float* const to_partial = a.partial + (static_cast<int64_t>(deal.slot * c.n_heads + g) * a.row_tiles + tile) * TILE * dim;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        float* const s = s_sum[n & 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // (16 bytes at a time, their places exchanged so that neither side has bank conflicts)
            const f32x4_t x = {acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]};
            *reinterpret_cast<f32x4_t*>(s + wk * CHUNK_WORDS + 4 * (i * 64 + (lane_e ^ (2 * i + 8 * half_e)))) = x;
        }
        __syncthreads();
        constexpr int FOURS = CHUNK_WORDS / 4;
#pragma unroll
        for (int r = 0; r < (FOURS + T - 1) / T; ++r) {  // four dims per lane, eight lanes together the 32 of a row
            const int four = tid_e + r * T, i = four & 3, h = (four >> 2) & 1, row = four >> 3, mr = m0 + row, d = 32 * n + 16 * h + 4 * i;
            if (four < FOURS && mr < n_pairs_rows && d < dim) {
                f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    x += *reinterpret_cast<const f32x4_t*>(s + w * CHUNK_WORDS + 4 * (i * 64 + ((32 * h + row) ^ (2 * i + 8 * h))));
                }
                if (partial) {
                    *reinterpret_cast<f32x4_t*>(to_partial + static_cast<int64_t>(row) * dim + d) = x;
                } else {
                    const int ir = div_small(mr, ratio);
                    const int64_t at = ((q0 + ir) * a.n_heads_q + g * ratio + (mr - ir * ratio)) * static_cast<int64_t>(dim) + d;
                    *reinterpret_cast<u32x2_t*>(out + at) = u32x2_t{pack2<Tag>(x[0] * a.c_out, x[1] * a.c_out), pack2<Tag>(x[2] * a.c_out, x[3] * a.c_out)};
                }
            }
        }
    }
}

}  // namespace hstu
