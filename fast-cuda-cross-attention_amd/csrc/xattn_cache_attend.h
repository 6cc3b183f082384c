// Attention over a paged cache, with or without a prefix that the whole batch
// shares: o = sum_c e^(s_c - m) v_c / sum_c e^(s_c - m), s_c = scale q.k_c, in one
// pass over the keys with the running maximum m.
//
// The query heads of one kv head see the same keys, so a sequence's rows are
// its (token, head of the group) pairs, `group` to a token.  A work item is
// (kv head, a tile of rows, a range of keys) on one workgroup of four wavefronts, in
// one of four forms: xattn_cache_few.h and xattn_cache_tile.h (16 bits up to dim 256),
// xattn_cache_ring.h (16 bits at 768), xattn_cache_wide.h (32 bits).
// Where there are fewer items than the device needs, the keys are divided and a
// second launch merges the parts.  For the prefix the rows are those of the whole
// batch, so that its keys are read once for a tile of rows of any sequences.
//
// Keys beyond the last row's reach are read from the last key within it, so that
// nothing is read that no row sees; keys that some rows of a tile do not see get
// the weight zero there.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "xattn_cache_few.h"
#include "xattn_cache_ring.h"
#include "xattn_cache_tile.h"
#include "xattn_cache_wide.h"
#include "xattn_launch.h"

namespace xattn {
namespace cache {

// --------------------------------------------------------------------------
// Kernels.  The keys of a prefix and those of the sequences are worked on in
// one launch, the prefix's (longer) items first: the sequences' fill in.
// --------------------------------------------------------------------------

// The forms by type and dim: that of a few rows (one block of sixteen), and that of
// many.  In 32 bits two blocks pay at 128 only: 1,024 tokens over 1,500 keys took
// 101 us with two and 120 with one there, but 69 and 62 at 64, 158 and 122 at 256, 79
// and 66 (512 tokens) at 768, where two leave too few registers or workgroups.
template <typename T, int D>
struct Forms {
    static constexpr bool kWide = sizeof(T) == 4, kRing = !kWide && D > 256;
    static constexpr bool kMany = !kWide || D == 128;
    // Rows of a work item of many, and the rows of a sequence from which on it is taken.
    static constexpr int kHeight = kWide || kRing ? 2 * kRows : TileShape<D>::kRows;
    static constexpr int kFrom = kWide || kRing ? kRows + 1 : 2 * kRows + 1;
    // Keys of a tile of the two, over all wavefronts.
    static constexpr int kFewKeys = kWide  ? WideShape<D, 1>::kKeys * kWaves / WideShape<D, 1>::kCols
                                    : kRing ? RingShape<1>::kKeys
                                            : FewShape<T, D>::kKeys * kWaves;
    static constexpr int kManyKeys = kWide || kRing ? kFewKeys : TileShape<D>::kKeys;
    static constexpr int lds(bool many) {
        if constexpr (kWide)
            return many ? WideShape<D, 2>::kLds : WideShape<D, 1>::kLds;
        else if constexpr (kRing)
            return many ? RingShape<2>::kLds : RingShape<1>::kLds;
        else
            return many ? TileShape<D>::kLds : FewShape<T, D>::kLds;
    }
    static constexpr int max_lds(bool a, bool b) { return lds(a) > lds(b) ? lds(a) : lds(b); }
    // Wavefronts that a SIMD has to hold: two of tile_item, in 256 registers each.
    static constexpr int waves(bool many) { return !kWide && !kRing && many ? 2 : 1; }
    // Workgroups of tile_item that a CU holds.
    static constexpr int kResident = D == 64 ? 3 : 2;
    template <bool MANY, bool PREFIX>
    static __device__ __forceinline__ void item(const AttendParams& p, unsigned block, char* lds) {
        if constexpr (kWide)
            wide_item<D, MANY ? 2 : 1, PREFIX>(p, block, lds);
        else if constexpr (kRing)
            ring_item<T, MANY ? 2 : 1, PREFIX>(p, block, lds);
        else if constexpr (MANY)
            tile_item<T, D, PREFIX>(p, block, lds);
        else
            attend_item<T, D, PREFIX>(p, block, lds);
    }
};

template <typename T, int D, bool MANY>
__global__ __launch_bounds__(256, (Forms<T, D>::waves(MANY))) void
cache_attend_kernel(AttendParams p) {
    __shared__ __align__(16) char lds[Forms<T, D>::lds(MANY)];
    Forms<T, D>::template item<MANY, false>(p, blockIdx.x, lds);
}

// PREFIX_MANY, MANY: the forms of the prefix's items and of the sequences'.
template <typename T, int D, bool PREFIX_MANY, bool MANY>
__global__ __launch_bounds__(256, (PREFIX_MANY && (MANY || D <= 128) ? Forms<T, D>::waves(true)
                                                                     : 1)) void
cache_prefix_kernel(AttendParams prefix, AttendParams own, unsigned prefix_blocks) {
    __shared__ __align__(16) char lds[Forms<T, D>::max_lds(PREFIX_MANY, MANY)];
    if (blockIdx.x < prefix_blocks)
        Forms<T, D>::template item<PREFIX_MANY, true>(prefix, blockIdx.x, lds);
    else
        Forms<T, D>::template item<MANY, false>(own, blockIdx.x - prefix_blocks, lds);
}

// --------------------------------------------------------------------------
// cache_merge_kernel: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the
// parts of a row.  LANES lanes take 256 columns of a row, or all of them.  Few
// rows of many parts (TOGETHER): a workgroup a row, its groups of LANES lanes taking
// every so many-th part.  Otherwise a group a row, those of a wavefront heads of
// one token: what a row waits for are four reads one after another (its sequence,
// length, maxima, parts), so many rows have to wait at once (26,076 rows of up to
// four parts of 64: 13.0 us with a wavefront a row, 7.4 with a group).
// --------------------------------------------------------------------------
template <int D>
struct MergeShape {
    static constexpr int kCols = D > 256 ? 256 : D, kLanes = kCols / 4;
    static constexpr int kGroups = kWave / kLanes;
    // Wavefronts of a call, workgroups if TOGETHER.
    static long long units(int tokens, int heads, bool together) {
        const int per = together ? 1 : kGroups;
        return (long long)tokens * (D / kCols) * ((heads + per - 1) / per);
    }
};

template <typename T, int D, bool TOGETHER>
__global__ __launch_bounds__(256) void cache_merge_kernel(AttendParams p, int prefix_parts) {
    typedef MergeShape<D> S;
    constexpr int COLS = S::kCols, LANES = S::kLanes, GROUPS = S::kGroups;
    constexpr int PER = TOGETHER ? 1 : GROUPS;          // rows of a wavefront
    constexpr int SHARE = kWave / PER;                  // lanes that share a row
    constexpr int STEP = TOGETHER ? GROUPS * kWaves : 1;
    __shared__ f4 sums[kWaves - 1][LANES];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, group = lane / LANES;
    const unsigned by_token = (p.heads + PER - 1) / PER * (D / COLS);
    const unsigned unit = TOGETHER ? blockIdx.x : blockIdx.x * kWaves + wave;
    const unsigned t0 = unit / by_token, rest = unit % by_token;
    if (t0 >= (unsigned)p.batch.tokens) return;
    const int t = __builtin_amdgcn_readfirstlane((int)t0);
    const int heads0 = (int)(rest / (D / COLS)) * PER + (TOGETHER ? 0 : group);
    const int head = min(heads0, p.heads - 1), col = (int)(rest % (D / COLS)) * COLS + lane % LANES * 4;
    const int b = token_sequence(p.batch, t);
    if (b >= p.batch.batch) return;
    const Sequence s = sequence(p.batch, b);
    if (t < s.first || t >= s.end) return;
    const int n = s.seen(t, p.causal);
    if (p.slot == 0 && (p.splits == 1 || n <= p.chunk)) return;  // stored already
    const int own = min((n + p.chunk - 1) / p.chunk, p.splits);
    const int parts = prefix_parts + own, me = lane % SHARE;
    const size_t at = ((size_t)t * p.heads + head) * p.slots;
    float top = -INFINITY;
    for (int i = me; i < parts; i += SHARE) top = fmaxf(top, p.ml[at + i].x);
#pragma unroll
    for (int o = 1; o < SHARE; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f4 x = {0, 0, 0, 0};
    const int first = TOGETHER ? group + wave * GROUPS : 0;
    for (int from = 0; from < parts; from += SHARE) {
        float weight = 0.0f;
        if (from + me < parts) {
            const float2 ml = p.ml[at + from + me];
            weight = fast_exp2(ml.x - ref);
            sum += weight * ml.y;
        }
        const int count = min(SHARE, parts - from);
#pragma unroll 4
        for (int i = first; i - first < count; i += STEP) {
            const int one = min(i, count - 1);
            const float w = __shfl(weight, lane - me + one);
            const f4 part = *(const f4*)(p.po + (at + from + one) * D + col);
            if (i < count) x += w * part;
        }
    }
#pragma unroll
    for (int o = 1; o < SHARE; o *= 2) sum += __shfl_xor(sum, o);
    if (s.bad) sum = NAN;
    if constexpr (TOGETHER) {
#pragma unroll
        for (int o = LANES; o < kWave; o *= 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o);
        if (wave > 0 && lane < LANES) sums[wave - 1][lane] = x;
        __syncthreads();
        if (wave > 0 || lane >= LANES) return;
#pragma unroll
        for (int w = 0; w + 1 < kWaves; ++w) x += sums[w][lane];
    }
    if (heads0 < p.heads) {
        Piece4<T> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.e[e] = (T)(x[e] / sum);
        *(Piece4<T>*)((T*)p.out + t * p.os + (long long)head * D + col) = y;
    }
}

// --------------------------------------------------------------------------
// Plan
// --------------------------------------------------------------------------
struct Range {
    int splits, chunk;
};
constexpr int kMaxSplits = 256;

// `keys` keys in about `s` ranges, each of whole `step` keys.  deal > 0: of a number
// that lets the streams of `deal` kv heads deal onto the XCDs (find_item).
static Range ranges(long long s, int keys, int step, int deal) {
    s = std::max<long long>(1, std::min<long long>(std::min(s, (long long)kMaxSplits), keys / step));
    if (deal > 0) {
        int by = kNumXcd;
        while (by > 1 && (long long)deal * by / 2 % kNumXcd == 0) by /= 2;
        if (s > by) s -= s % by;
    }
    long long chunk = (keys + s - 1) / s;
    chunk = std::max<long long>(step, (chunk + step - 1) / step * step);
    if (deal == 0) s = std::max<long long>(1, (keys + chunk - 1) / chunk);
    return {(int)s, (int)chunk};
}

struct Plan {
    bool single;                 // every sequence has one row tile
    bool many, prefix_many;      // the forms
    int tiles, prefix_tiles;     // row tiles
    Range own, prefix;
    int slots() const { return own.splits + prefix.splits; }
    int prefix_parts(int len) const {
        return std::min(prefix.splits, (int)((len + (long long)prefix.chunk - 1) / prefix.chunk));
    }
};

// How often the keys are divided.
//   One row tile to a sequence: enough for a workgroup a CU, and so that none has
// more than 1 MiB of K and V to read (3 at dim 768, where a workgroup has a CU to
// itself), as sequences may be of unlike lengths: 64 of up to 8,192 keys, 8 kv heads
// of 128, take 214 us in ranges of 1 MiB, 232 in ranges of 2.  Up to 256 KiB stay
// whole even on an idle device: 784 keys of 64 take 9.7 us whole and 13.4 in seven
// parts with the merge, 3,000 take 20.8 and 12.6.
//   Several row tiles: a workgroup a CU; of tile_item as many as the device holds at
// once.  (12 heads on 4 kv heads of 128: six pieces of 400 tokens over 4,000 keys take
// 101, 87, 105 and 97 us in 1, 2, 3 and 4 ranges, 2 being what it holds; 32 on 8: one
// of 500 over 6,000 keys 142, 87, 80, 72, 86 in 1 .. 5, 4 being it.)
//   The prefix: a workgroup a CU (32 tokens over 16,384 keys, 8 kv heads of 128: 37
// us, 46 with two, 50 with three: more parts to merge).
template <typename T, int D>
static Plan plan(const Attention& a) {
    typedef Forms<T, D> F;
    constexpr long long row = 2LL * D * sizeof(T);  // bytes of a key and its value
    Plan p;
    const int kv = (int)a.pages.kv_heads, group = a.heads / kv;
    const long long rows = (long long)a.batch.tokens * group, most = (long long)a.max_q * group;
    const long long cu = device_cu_count();
    constexpr bool tile = !F::kWide && !F::kRing;
    // Two blocks instead of one pay where a CU has many keys to pass them by, as every
    // range has a start and a tail: in 16 bits at 768, 64 rows over 16,000 keys take 42
    // us with two and 36 with one, over 50,176 keys 69 and 79; in 32 bits at 128, 256
    // rows of 8 kv heads over 784 keys 25 and 22, 2,048 over 1,500 keys 101 and 119.
    const long long passes = std::min(rows / kRows + a.batch.batch,
                                      (most + kRows - 1) / kRows * a.batch.batch) * a.max_kv +
                             rows / kRows * a.prefix_len;
    const bool enough = tile || passes * kv >= (F::kRing ? 512 : 1024) * cu;
    p.many = F::kMany && enough && most >= F::kFrom;
    const int height = p.many ? F::kHeight : kRows;
    p.single = most <= height;
    p.tiles = p.single ? a.batch.batch
                       : (int)std::min<long long>(rows / height + a.batch.batch,
                                                  (most + height - 1) / height * a.batch.batch);
    const long long items = std::max<long long>(1, (long long)p.tiles * kv);
    long long s = (tile && p.many && !p.single ? F::kResident : 1) * cu / items;
    if (p.single) {
        const long long by_size = a.max_kv * row / ((D > 256 ? 3LL : 1LL) << 20);
        s = std::max(s, std::min(by_size, 16 * cu / items));
        if (a.max_kv * row <= 256 << 10) s = 1;
    }
    const auto divide = [&](long long s, int keys, bool many, bool deal) {
        // where tile_item works, its matrix instructions bound it, not what L2 misses
        return tile && many ? ranges(s, keys, 2 * F::kManyKeys, 0)
                            : ranges(s, keys, F::kFewKeys, deal ? kv : 0);
    };
    p.own = divide(s, a.max_kv, p.many, !p.single);
    p.prefix_many = F::kMany && enough && rows >= F::kFrom;
    const int prefix_height = p.prefix_many ? F::kHeight : kRows;
    p.prefix_tiles = (int)((rows + prefix_height - 1) / prefix_height);
    p.prefix = Range{0, 1};
    if (a.prefix_len > 0)
        p.prefix = divide(cu / std::max<long long>(1, (long long)p.prefix_tiles * kv),
                          a.prefix_len, p.prefix_many, true);
    return p;
}

static size_t parts(const Attention& a, const Plan& p) {
    if (p.prefix.splits == 0 && p.own.splits == 1) return 0;
    return (size_t)a.batch.tokens * a.heads * p.slots();
}

// Workgroups of the launches: the prefix's, those and the sequences' own, the merge's.
struct Grid {
    long long first, all, merge;
    bool together;
};

template <int D>
static Grid grid(const Attention& a, const Plan& plan) {
    const long long kv = a.pages.kv_heads;
    Grid g;
    g.first = kv * plan.prefix_tiles * plan.prefix.splits;
    g.all = g.first + kv * plan.tiles * plan.own.splits;
    g.together = MergeShape<D>::units(a.batch.tokens, a.heads, true) < 8 * device_cu_count();
    const long long units = MergeShape<D>::units(a.batch.tokens, a.heads, g.together);
    g.merge = parts(a, plan) == 0 ? 0 : g.together ? units : (units + kWaves - 1) / kWaves;
    return g;
}

template <typename T, int D>
static void go(const Attention& a, const Plan& plan, void* scratch, hipStream_t stream) {
    typedef Forms<T, D> F;
    AttendParams own{};
    own.pages = a.pages;
    own.batch = a.batch;
    own.prefix_pages = a.prefix_pages;
    own.prefix_len = a.prefix_len;
    own.heads = a.heads;
    own.group = FastDiv::of((unsigned)a.heads / a.pages.kv_heads);
    own.q = a.q;
    own.out = a.out;
    own.qs = a.qs;
    own.os = a.os;
    // A scale of zero makes all scores equal; so does one that is next to it, and a
    // masked score's -infinity stays one.
    own.c2 = std::max(std::fabs(a.scale) * kLog2e, 1e-37f);
    own.lag = std::min(kLag / own.c2, 1e30f);
    own.sign = a.scale >= 0 ? 0 : a.dtype == XATTN_F32 ? 0x80000000u : 0x80008000u;
    own.causal = a.causal;
    own.tiles = plan.tiles;
    own.single = plan.single;
    own.splits = plan.own.splits;
    own.chunk = plan.own.chunk;
    own.slot = plan.prefix_parts(a.prefix_len);
    own.slots = plan.slots();
    if (const size_t n = parts(a, plan)) {
        own.po = (float*)scratch;
        own.ml = (float2*)(own.po + n * D);
    }
    const Grid g = grid<D>(a, plan);
    if (!grid_fits("cache attention", std::max(g.all, g.merge))) return;
    const unsigned first = (unsigned)g.first, all = (unsigned)g.all;
    if (first > 0) {
        AttendParams p = own;
        p.single = 0;
        p.tiles = plan.prefix_tiles;
        p.splits = plan.prefix.splits;
        p.chunk = plan.prefix.chunk;
        p.slot = 0;
        // a sequence has no more rows than the batch
        if constexpr (F::kMany) {
            if (plan.many)
                cache_prefix_kernel<T, D, true, true><<<all, 256, 0, stream>>>(p, own, first);
            else if (plan.prefix_many)
                cache_prefix_kernel<T, D, true, false><<<all, 256, 0, stream>>>(p, own, first);
        }
        if (!plan.prefix_many)
            cache_prefix_kernel<T, D, false, false><<<all, 256, 0, stream>>>(p, own, first);
    } else if (!plan.many) {
        cache_attend_kernel<T, D, false><<<all, 256, 0, stream>>>(own);
    } else {
        if constexpr (F::kMany) cache_attend_kernel<T, D, true><<<all, 256, 0, stream>>>(own);
    }
    const unsigned merge = (unsigned)g.merge;
    if (merge > 0 && g.together)
        cache_merge_kernel<T, D, true><<<merge, 256, 0, stream>>>(own, own.slot);
    else if (merge > 0)
        cache_merge_kernel<T, D, false><<<merge, 256, 0, stream>>>(own, own.slot);
}

// f(T{}, dim as a constant) for the call's type and dim.
template <typename F>
static void dispatch(const Attention& a, F f) {
    const auto by_dim = [&](auto type) {
        if (a.pages.dim == 64) f(type, std::integral_constant<int, 64>{});
        if (a.pages.dim == 128) f(type, std::integral_constant<int, 128>{});
        if (a.pages.dim == 256) f(type, std::integral_constant<int, 256>{});
        if (a.pages.dim == kDim) f(type, std::integral_constant<int, kDim>{});
    };
    if (a.dtype == XATTN_F32) by_dim(float{});
    if (a.dtype == XATTN_F16) by_dim(_Float16{});
    if (a.dtype == XATTN_BF16) by_dim(__bf16{});
}

size_t attention_scratch(const Attention& a) {
    size_t n = 0;
    dispatch(a, [&](auto type, auto dim) {
        constexpr int D = dim();
        const Plan p = plan<decltype(type), D>(a);
        const Grid g = grid<D>(a, p);
        if (std::max(g.all, g.merge) <= kMaxBlocks)  // else the launch refuses
            n = parts(a, p) * (D * sizeof(float) + sizeof(float2));
    });
    return n;
}

bool launch_attention(const Attention& a, void* scratch, hipStream_t stream) {
    dispatch(a, [&](auto type, auto dim) {
        typedef decltype(type) T;
        go<T, dim()>(a, plan<T, dim()>(a), scratch, stream);
    });
    return check_launch("cache attention");
}

}  // namespace cache
}  // namespace xattn
