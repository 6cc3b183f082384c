// Attention over a paged cache, with or without a prefix that the whole batch
// shares: o = sum_c e^(s_c - m) v_c / sum_c e^(s_c - m), s_c = scale q.k_c, in one
// pass over the keys with the running maximum m.
//
// The query heads of one kv head see the same keys, so a sequence's rows are
// its (token, head of the group) pairs, `group` to a token.  A work item is
// (kv head, a tile of rows, a range of keys) on one workgroup of four wavefronts, in
// one of three forms: xattn_cache_few.h, xattn_cache_ring.h, xattn_cache_tile.h.
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

#include "xattn_cache_few.h"
#include "xattn_cache_ring.h"
#include "xattn_cache_tile.h"
#include "xattn_launch.h"

namespace xattn {
namespace cache {

#ifndef WANT_TILE
#define WANT_TILE 6
#define WANT_FEW 1
#define WANT_SINGLE 8
#define WANT_PREFIX 1
#define TILE_STEP 2
#endif
// --------------------------------------------------------------------------
// Kernels.  The keys of a prefix and those of the sequences are worked on in
// one launch, the prefix's (longer) items first: the sequences' fill in.
// --------------------------------------------------------------------------
// Which form takes a few rows: attend_item in 16 bits up to dim 256, else ring_item.
template <typename T, int D>
constexpr bool kRing = sizeof(T) == 4 || D > 256;
template <typename T, int D>
constexpr int few_lds() {
    if constexpr (kRing<T, D>)
        return RingShape<T, D>::kLds;
    else
        return FewShape<T, D>::kLds;
}
template <typename T, int D, bool PREFIX>
__device__ __forceinline__ void few_item(const AttendParams& p, unsigned block, char* lds) {
    if constexpr (kRing<T, D>)
        ring_item<T, D, PREFIX>(p, block, lds);
    else
        attend_item<T, D, PREFIX>(p, block, lds);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void cache_attend_kernel(AttendParams p) {
    __shared__ __align__(16) char lds[few_lds<T, D>()];
    few_item<T, D, false>(p, blockIdx.x, lds);
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void cache_tile_kernel(AttendParams p) {
    __shared__ __align__(16) char lds[TileShape<D>::kLds];
    tile_item<T, D, false>(p, blockIdx.x, lds);
}

// TILES: how many of the two go by tile_item (2: both, 1: the prefix, 0: none).
template <typename T, int D, int TILES>
__global__ __launch_bounds__(256, TILES == 2 || (TILES == 1 && D <= 128) ? 2 : 1) void
cache_prefix_kernel(
    AttendParams prefix, AttendParams own, unsigned prefix_blocks) {
    constexpr int few = TILES < 2 ? few_lds<T, D>() : 0;
    constexpr int many = TILES > 0 ? TileShape<D>::kLds : 0;
    __shared__ __align__(16) char lds[few > many ? few : many];
    if (blockIdx.x < prefix_blocks) {
        if constexpr (TILES > 0)
            tile_item<T, D, true>(prefix, blockIdx.x, lds);
        else
            few_item<T, D, true>(prefix, blockIdx.x, lds);
    } else {
        if constexpr (TILES > 1)
            tile_item<T, D, false>(own, blockIdx.x - prefix_blocks, lds);
        else
            few_item<T, D, false>(own, blockIdx.x - prefix_blocks, lds);
    }
}

// --------------------------------------------------------------------------
// cache_merge_kernel: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the
// parts of a row.  A wavefront takes 256 columns of a row, or all of them, in
// 64 / LANES groups of LANES lanes that take every so many-th part; with
// `together` the four wavefronts of a workgroup share a row's parts (few rows of
// many parts), otherwise each has a row of its own.
// --------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_merge_kernel(AttendParams p, int prefix_parts,
                                                          int together) {
    constexpr int COLS = D > 256 ? 256 : D, LANES = COLS / 4, GROUPS = kWave / LANES;
    __shared__ f4 sums[kWaves - 1][LANES];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const unsigned unit = together ? blockIdx.x : blockIdx.x * kWaves + wave;
    const unsigned row = unit / (D / COLS), col = unit % (D / COLS) * COLS + lane % LANES * 4;
    const int t = (int)(row / p.heads), head = (int)(row % p.heads);
    if (t >= p.batch.tokens) return;
    const int b = token_sequence(p.batch, t);
    if (b >= p.batch.batch) return;
    const Sequence s = sequence(p.batch, b);
    if (t < s.first || t >= s.end) return;
    const int n = s.seen(t, p.causal);
    if (p.slot == 0 && (p.splits == 1 || n <= p.chunk)) return;  // stored already
    const int own = min((n + p.chunk - 1) / p.chunk, p.splits);
    const int parts = prefix_parts + own;
    const size_t at = (size_t)row * p.slots;
    float top = -INFINITY;
    for (int i = lane; i < parts; i += kWave) top = fmaxf(top, p.ml[at + i].x);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f4 x = {0, 0, 0, 0};
    const int first = lane / LANES + (together ? wave * GROUPS : 0);
    const int step = GROUPS * (together ? kWaves : 1);
    for (int from = 0; from < parts; from += kWave) {
        float weight = 0.0f;
        if (from + lane < parts) {
            const float2 ml = p.ml[at + from + lane];
            weight = fast_exp2(ml.x - ref);
            sum += weight * ml.y;
        }
        const int count = min(kWave, parts - from);
#pragma unroll 4
        for (int i = first; i - first < count; i += step) {
            const int one = min(i, count - 1);
            const float w = __shfl(weight, one);
            const f4 part = *(const f4*)(p.po + (at + from + one) * D + col);
            if (i < count) x += w * part;
        }
    }
    sum = wave_sum(sum);
    if (s.bad) sum = NAN;
#pragma unroll
    for (int o = LANES; o < kWave; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o);
    if (together) {
        if (wave > 0 && lane < LANES) sums[wave - 1][lane] = x;
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 0; w + 1 < kWaves; ++w) x += sums[w][lane % LANES];
    }
    if (lane < LANES) {
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
constexpr int kManyRows = 32;  // rows of a sequence beyond which tile_item takes it

// Ranges that `keys` keys are divided into where all of them are `items` items of
// work: as many as make `want` workgroups, each of `step` keys or more; with
// several row tiles to a range, of a number that lets the streams deal onto
// the XCDs (find_item).
static Range ranges(long long items, int keys, int step, long long want, int kv, bool single) {
    long long s = std::min<long long>(items > 0 ? want / items : 1, keys / step);
    s = std::max<long long>(1, std::min<long long>(s, kMaxSplits));
    int deal = kNumXcd;
    while (deal > 1 && (long long)kv * deal / 2 % kNumXcd == 0) deal /= 2;
    if (!single && s > deal) s -= s % deal;
    long long chunk = (keys + s - 1) / s;
    chunk = std::max<long long>(step, (chunk + step - 1) / step * step);
    return {single ? (int)std::max<long long>(1, (keys + chunk - 1) / chunk) : (int)s, (int)chunk};
}

struct Plan {
    bool single;            // every sequence has at most sixteen rows
    int rows, prefix_rows;  // rows of a work item
    int tiles, prefix_tiles;
    Range own, prefix;
    int slots() const { return own.splits + prefix.splits; }
    int prefix_parts(int len) const {
        return std::min(prefix.splits, (int)((len + (long long)prefix.chunk - 1) / prefix.chunk));
    }
};

static int tile_rows(int dim) { return dim > 128 ? TileShape<256>::kRows : TileShape<128>::kRows; }

static Plan plan(const Attention& a) {
    Plan p;
    const int kv = (int)a.pages.kv_heads, group = a.heads / kv, dim = a.pages.dim;
    const bool tiled = a.dtype != XATTN_F32 && dim <= 256;  // tile_item takes it
    const int few = (a.dtype == XATTN_F32 ? 16 : 32) * (dim > 256 ? 1 : kWaves);
    const int many = dim > 128 ? TileShape<256>::kKeys : TileShape<128>::kKeys;
    const long long rows = (long long)a.batch.tokens * group, most = (long long)a.max_q * group;
    const long long cu = device_cu_count();
    p.single = most <= kRows;
    p.rows = tiled && most > kManyRows ? tile_rows(dim) : kRows;
    p.tiles = p.single ? a.batch.batch
                       : (int)std::min<long long>(rows / p.rows + a.batch.batch,
                                                  (most + p.rows - 1) / p.rows * a.batch.batch);
    p.own = ranges((long long)p.tiles * kv, a.max_kv, p.rows > kRows ? TILE_STEP * many : few,
                   p.single ? WANT_SINGLE * cu : p.rows > kRows ? WANT_TILE * cu : WANT_FEW * cu, kv, p.single);
    p.prefix_rows = tiled && rows > kManyRows ? tile_rows(dim) : kRows;
    p.prefix_tiles = (int)((rows + p.prefix_rows - 1) / p.prefix_rows);
    p.prefix = a.prefix_len > 0
                   ? ranges((long long)p.prefix_tiles * kv, a.prefix_len,
                            p.prefix_rows > kRows ? TILE_STEP * many : few, WANT_PREFIX * cu, kv, false)
                   : Range{0, 1};
    return p;
}

static size_t parts(const Attention& a, const Plan& p) {
    if (p.prefix.splits == 0 && p.own.splits == 1) return 0;
    return (size_t)a.batch.tokens * a.heads * p.slots();
}

size_t attention_scratch(const Attention& a) {
    return parts(a, plan(a)) * (a.pages.dim * sizeof(float) + sizeof(float2));
}

static unsigned blocks(const AttendParams& p) {
    return p.pages.kv_heads * (unsigned)p.tiles * (unsigned)p.splits;
}

template <typename T, int D>
static void go(const AttendParams& own, const Plan& plan, hipStream_t stream) {
    constexpr bool tiled = sizeof(T) == 2 && D <= 256;
    const bool tile = tiled && plan.rows > kRows, prefix_tile = tiled && plan.prefix_rows > kRows;
    if (plan.prefix.splits > 0) {
        AttendParams p = own;
        p.single = 0;
        p.tiles = plan.prefix_tiles;
        p.splits = plan.prefix.splits;
        p.chunk = plan.prefix.chunk;
        p.slot = 0;
        const unsigned first = blocks(p), all = first + blocks(own);
        if constexpr (tiled) {
            if (tile)
                cache_prefix_kernel<T, D, 2><<<all, 256, 0, stream>>>(p, own, first);
            else if (prefix_tile)
                cache_prefix_kernel<T, D, 1><<<all, 256, 0, stream>>>(p, own, first);
        }
        if (!prefix_tile) cache_prefix_kernel<T, D, 0><<<all, 256, 0, stream>>>(p, own, first);
    } else if (tile) {
        if constexpr (tiled) cache_tile_kernel<T, D><<<blocks(own), 256, 0, stream>>>(own);
    } else {
        cache_attend_kernel<T, D><<<blocks(own), 256, 0, stream>>>(own);
    }
    if (own.po) {
        const long long units = (long long)own.batch.tokens * own.heads * (D > 256 ? D / 256 : 1);
        const bool together = units < 8 * device_cu_count();
        cache_merge_kernel<T, D>
            <<<(unsigned)(together ? units : (units + kWaves - 1) / kWaves), 256, 0, stream>>>(
                own, own.slot, together);
    }
}

template <typename T>
static void by_dim(AttendParams& p, const Plan& plan, hipStream_t stream) {
    if (p.pages.dim == 64) go<T, 64>(p, plan, stream);
    if (p.pages.dim == 128) go<T, 128>(p, plan, stream);
    if (p.pages.dim == 256) go<T, 256>(p, plan, stream);
    if (p.pages.dim == kDim) go<T, kDim>(p, plan, stream);
}

bool launch_attention(const Attention& a, void* scratch, hipStream_t stream) {
    const Plan pl = plan(a);
    AttendParams p{};
    p.pages = a.pages;
    p.batch = a.batch;
    p.prefix_pages = a.prefix_pages;
    p.prefix_len = a.prefix_len;
    p.heads = a.heads;
    p.group = FastDiv::of((unsigned)a.heads / a.pages.kv_heads);
    p.q = a.q;
    p.out = a.out;
    p.qs = a.qs;
    p.os = a.os;
    // A scale of zero makes all scores equal; so does one that is next to it, and a
    // masked score's -infinity stays one.
    p.c2 = std::max(std::fabs(a.scale) * kLog2e, 1e-37f);
    p.lag = std::min(kLag / p.c2, 1e30f);
    p.sign = a.scale >= 0 ? 0 : a.dtype == XATTN_F32 ? 0x80000000u : 0x80008000u;
    p.causal = a.causal;
    p.tiles = pl.tiles;
    p.single = pl.single;
    p.splits = pl.own.splits;
    p.chunk = pl.own.chunk;
    p.slot = pl.prefix_parts(a.prefix_len);
    p.slots = pl.slots();
    if (const size_t n = parts(a, pl)) {
        p.po = (float*)scratch;
        p.ml = (float2*)(p.po + n * a.pages.dim);
    }
    if (a.dtype == XATTN_F32) by_dim<float>(p, pl, stream);
    if (a.dtype == XATTN_F16) by_dim<_Float16>(p, pl, stream);
    if (a.dtype == XATTN_BF16) by_dim<__bf16>(p, pl, stream);
    return check_launch("cache_attend_kernel");
}

}  // namespace cache
}  // namespace xattn
