// Rotary positions, and keys and values appended to a paged cache with the
// rotation on the way.
//
// Pair i of a head at position p turns by the angle a = 2 pi p f_i:
//     (x, y) -> (x c - y s, y c + x s),  c = A cos a,  s = A sin a
// (the gradient takes -s: the transpose).  p f_i is formed in 64 bits as turns
// and its whole turns are dropped before it goes to 32, so the angle is good to
// 2^-25 of a turn at any position.
//
// Both kernels are bound by memory: about 6 operations for each 2 to 4 bytes
// moved (4.8 TB/s rotating 8,192 tokens of 32 heads of 128 in 16 bits, 4.1 appending
// 8,965 of 8; a copy of 2 GB runs at 4.8).  A workgroup takes a few tokens; it first puts their cosines and
// sines in LDS, each once for all of the token's heads, and then moves the
// heads in 16-byte pieces, both halves of a pair in one thread, so that y may
// be x.
#pragma once

#include <algorithm>

#include "xattn_cache.h"
#include "xattn_launch.h"

namespace xattn {
namespace cache {

constexpr int kThreads = 256;
constexpr int kMaxAngles = kMaxRot / 2;  // cosines and sines of a workgroup's tokens (8 KiB of LDS)
constexpr int kMaxTokens = 64;           // tokens of a workgroup

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
    T e[V];
};

// One head's part of the work: `units` units of V elements (pairs of V for
// the rotated ones of the half layout, V / 2 pairs for the interleaved one;
// with V = 1 always one pair), in the order rotated, then copied.
template <typename T, int V, bool IL>
struct Head {
    static __host__ __device__ int rotated(int rot) {
        return IL ? (V == 1 ? rot / 2 : rot / V) : rot / 2 / V;
    }
    static __host__ __device__ int units(int dim, int rot) {
        return rotated(rot) + (dim - rot) / V;
    }
    // cs: (cos, sin) of the token's pairs.
    static __device__ void unit(const T* x, T* y, int u, int rot, const float2* cs) {
        typedef Piece<T, V> P;
        const int nr = rotated(rot);
        if (u >= nr) {
            const int at = rot + (u - nr) * V;
            if (x != y) *(P*)(y + at) = *(const P*)(x + at);
            return;
        }
        if constexpr (IL) {
            constexpr int E = V == 1 ? 2 : V;
            const int at = u * E;
            T in[E];
            if constexpr (V == 1) {
                in[0] = x[at];
                in[1] = x[at + 1];
            } else {
                *(P*)in = *(const P*)(x + at);
            }
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 t = cs[(at + e) / 2];
                const float a = to_f32(in[e]), b = to_f32(in[e + 1]);
                in[e] = from_f32<T>(a * t.x - b * t.y);
                in[e + 1] = from_f32<T>(b * t.x + a * t.y);
            }
            if constexpr (V == 1) {
                y[at] = in[0];
                y[at + 1] = in[1];
            } else {
                *(P*)(y + at) = *(const P*)in;
            }
        } else {
            const int at = u * V;
            P p = *(const P*)(x + at), q = *(const P*)(x + at + rot / 2);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 t = cs[at + e];
                const float a = to_f32(p.e[e]), b = to_f32(q.e[e]);
                p.e[e] = from_f32<T>(a * t.x - b * t.y);
                q.e[e] = from_f32<T>(b * t.x + a * t.y);
            }
            *(P*)(y + at) = p;
            *(P*)(y + at + rot / 2) = q;
        }
    }
};

__device__ inline float2 angle(const Rope& R, int position, int i) {
    double turns = (double)position * R.freqs[i];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    return {c * R.amplitude, (R.inverse ? -s : s) * R.amplitude};
}

struct RopeParams {
    const void* x;
    void* y;
    const int* positions;
    Rope rope;
    int tokens, heads, dim, per;  // per: tokens of a workgroup
    long long xs, ys;
    FastDiv units, by_heads;
};

template <typename T, int V, bool IL>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams p) {
    __shared__ float2 cs[kMaxAngles];
    const int half = p.rope.rot / 2;
    const long long t0 = (long long)blockIdx.x * p.per;
    const int n = (int)min((long long)p.per, p.tokens - t0);
    for (int i = threadIdx.x; i < n * half; i += kThreads)
        cs[i] = angle(p.rope, p.positions[t0 + i / half], i % half);
    __syncthreads();
    const unsigned all = (unsigned)n * p.heads * p.units.d;
    for (unsigned i = threadIdx.x; i < all; i += kThreads) {
        const unsigned row = p.units.div(i), u = i - row * p.units.d;
        const unsigned t = p.by_heads.div(row), h = row - t * p.heads;
        const T* x = (const T*)p.x + (t0 + t) * p.xs + (long long)h * p.dim;
        T* y = (T*)p.y + (t0 + t) * p.ys + (long long)h * p.dim;
        Head<T, V, IL>::unit(x, y, (int)u, p.rope.rot, cs + t * half);
    }
}

struct AppendParams {
    Pages pages;
    Batch batch;
    Rope rope;
    const void* k;
    const void* v;
    const void* q;
    void* q_out;
    const int* positions;
    int heads, per;  // heads: query heads that are rotated too, or 0
    long long ks, vs, qs, qos;
    FastDiv units, copies, by_token;  // of a rotated head, of a copied one, of a token
};

template <typename T, int V, bool IL>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(AppendParams p) {
    __shared__ float2 cs[kMaxAngles];
    __shared__ int place[kMaxTokens];    // position to rotate by
    __shared__ int owned[kMaxTokens];    // the token has a sequence
    __shared__ int stored[kMaxTokens];   // ... and a slot:
    __shared__ unsigned row[kMaxTokens];  // its row of kv head 0
    const int half = p.rope.rot / 2, dim = p.pages.dim;
    const long long t0 = (long long)blockIdx.x * p.per;
    const int n = (int)min((long long)p.per, p.batch.tokens - t0);
    for (int i = threadIdx.x / kWave; i < n; i += kThreads / kWave) {
        const int t = (int)t0 + i, b = token_sequence(p.batch, t);
        int first = 0, end = 0, at = 0;
        bool own = false, has = false;
        unsigned r = 0;
        if (b < p.batch.batch) {
            sequence_rows(p.batch, b, &first, &end);
            own = t >= first && t < end;
        }
        if (own) {
            const long long pos =
                (long long)p.batch.kv_lens[b] - (p.batch.q_starts[b + 1] - t);
            at = (int)pos;
            if (pos >= 0 && pos < p.batch.capacity) {
                const unsigned page = p.pages.page_size.div((unsigned)pos);
                const unsigned slot = (unsigned)pos - page * p.pages.page_size.d;
                const int id = p.batch.page_table[(long long)b * p.batch.width + page];
                has = id >= 0 && (unsigned)id < p.pages.num_pages;
                r = (unsigned)id * p.pages.kv_heads * p.pages.page_size.d + slot;
            }
            if (p.positions) at = p.positions[t];
        }
        if (threadIdx.x % kWave == 0) {
            place[i] = at;
            owned[i] = own;
            stored[i] = has;
            row[i] = r;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * half; i += kThreads)
        cs[i] = angle(p.rope, place[i / half], i % half);
    __syncthreads();
    // A token's units: the query heads', the key heads', the value heads'.
    const unsigned turned = (unsigned)(p.heads + p.pages.kv_heads) * p.units.d;
    const unsigned all = (unsigned)n * p.by_token.d;
    for (unsigned i = threadIdx.x; i < all; i += kThreads) {
        const unsigned t = p.by_token.div(i), rem = i - t * p.by_token.d;
        if (!owned[t]) continue;
        const long long token = t0 + t;
        if (rem < turned) {
            unsigned h = p.units.div(rem);
            const unsigned u = rem - h * p.units.d;
            const T* x;
            T* y;
            if (h < (unsigned)p.heads) {
                x = (const T*)p.q + token * p.qs + (long long)h * dim;
                y = (T*)p.q_out + token * p.qos + (long long)h * dim;
            } else {
                if (!stored[t]) continue;
                h -= p.heads;
                x = (const T*)p.k + token * p.ks + (long long)h * dim;
                y = (T*)p.pages.k + (size_t)(row[t] + h * p.pages.page_size.d) * dim;
            }
            Head<T, V, IL>::unit(x, y, (int)u, p.rope.rot, cs + t * half);
        } else if (stored[t]) {
            const unsigned h = p.copies.div(rem - turned);
            const unsigned u = rem - turned - h * p.copies.d;
            typedef Piece<T, V> P;
            *(P*)((T*)p.pages.v + (size_t)(row[t] + h * p.pages.page_size.d) * dim + u * V) =
                *(const P*)((const T*)p.v + token * p.vs + (long long)h * dim + u * V);
        }
    }
}

// Tokens of a workgroup: enough for `each` units a thread, as many as their
// angles leave room for, and no more than leave two workgroups a CU.  (8,192
// tokens of 32 heads of 128, 134 MB: 29.0, 27.5, 28.2 and 35.4 us with 2, 4, 8 and 16
// units; 8,965 of 8 appended, 73 MB: 17.8, 19.8, 22.0 and 32.3, as there one
// workgroup's look-ups pass while others move.)
static int tokens_per_workgroup(int tokens, long long units, int half, int each) {
    long long n = each * kThreads / units;
    n = std::min<long long>(n, half ? kMaxAngles / half : kMaxTokens);
    n = std::min<long long>(n, tokens / (2 * device_cu_count()));
    return (int)std::max<long long>(1, std::min<long long>(n, kMaxTokens));
}

// Whether heads of dim elements, rot of them rotated, go in 16-byte pieces:
// every piece lies in one half of its head's rotated part, or behind it.
static bool in_pieces(int size, int dim, int rot, bool interleaved) {
    const int v = 16 / size;
    return dim % v == 0 && (interleaved ? rot : rot / 2) % v == 0;
}
static bool aligned(const void* p, long long stride, int size) {
    return (uintptr_t)p % 16 == 0 && stride * size % 16 == 0;
}

template <typename T, int V, bool IL>
static void go(RopeParams& p, hipStream_t stream) {
    typedef Head<T, V, IL> H;
    p.units = FastDiv::of(H::units(p.dim, p.rope.rot));
    p.by_heads = FastDiv::of(p.heads);
    p.per = tokens_per_workgroup(p.tokens, (long long)p.heads * p.units.d, p.rope.rot / 2, 4);
    const long long blocks = ((long long)p.tokens + p.per - 1) / p.per;
    if (grid_fits("rope_kernel", blocks))
        rope_kernel<T, V, IL><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
}

template <typename T, int V, bool IL>
static void go(AppendParams& p, hipStream_t stream) {
    typedef Head<T, V, IL> H;
    p.units = FastDiv::of(H::units(p.pages.dim, p.rope.rot));
    p.copies = FastDiv::of(p.pages.dim / V);
    p.by_token = FastDiv::of((p.heads + p.pages.kv_heads) * p.units.d +
                             p.pages.kv_heads * p.copies.d);
    p.per = tokens_per_workgroup(p.batch.tokens, p.by_token.d, p.rope.rot / 2, 2);
    const long long blocks = ((long long)p.batch.tokens + p.per - 1) / p.per;
    if (grid_fits("cache_append_kernel", blocks))
        cache_append_kernel<T, V, IL><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
}

template <typename T, typename P>
static void by_layout(P& p, bool pieces, hipStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    if (pieces)
        p.rope.interleaved ? go<T, V, true>(p, stream) : go<T, V, false>(p, stream);
    else
        p.rope.interleaved ? go<T, 1, true>(p, stream) : go<T, 1, false>(p, stream);
}

template <typename P>
static void by_type(P& p, int dtype, bool pieces, hipStream_t stream) {
    if (dtype == XATTN_F32) by_layout<float>(p, pieces, stream);
    if (dtype == XATTN_F16) by_layout<_Float16>(p, pieces, stream);
    if (dtype == XATTN_BF16) by_layout<__bf16>(p, pieces, stream);
}

bool launch_rope(const void* x, void* y, const int* positions, const Rope& rope, int dtype,
                 int tokens, int heads, int dim, long long xs, long long ys,
                 hipStream_t stream) {
    const int size = dtype == XATTN_F32 ? 4 : 2;
    RopeParams p{x, y, positions, rope, tokens, heads, dim, 1, xs, ys, {}, {}};
    by_type(p, dtype,
            in_pieces(size, dim, rope.rot, rope.interleaved) && aligned(x, xs, size) &&
                aligned(y, ys, size),
            stream);
    return check_launch("rope_kernel");
}

bool launch_append(const Pages& pages, const Batch& batch, const Rope& rope, int dtype,
                   const void* k, long long ks, const void* v, long long vs, const void* q,
                   long long qs, void* q_out, long long qos, int heads, const int* positions,
                   hipStream_t stream) {
    const int size = dtype == XATTN_F32 ? 4 : 2;
    AppendParams p{pages, batch, rope, k, v, q, q_out, positions, q ? heads : 0, 1,
                   ks, vs, qs, qos, {}, {}, {}};
    bool pieces = in_pieces(size, pages.dim, rope.rot, rope.interleaved) &&
                  aligned(k, ks, size) && aligned(v, vs, size);
    if (q) pieces = pieces && aligned(q, qs, size) && aligned(q_out, qos, size);
    by_type(p, dtype, pieces, stream);
    return check_launch("cache_append_kernel");
}

}  // namespace cache
}  // namespace xattn
