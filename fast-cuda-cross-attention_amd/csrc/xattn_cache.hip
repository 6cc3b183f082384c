// Attention over a paged cache, with or without a prefix that the whole batch
// shares: o = sum_c e^(s_c - m) v_c / sum_c e^(s_c - m), s_c = scale q.k_c, m the
// running maximum.
//
// One wavefront per (token, head), a lane holding dim / 64 consecutive
// elements of q, k, v and o; one pass over the keys.
#include "xattn_cache.h"
#include "xattn_launch.h"

namespace xattn {
namespace cache {

template <typename T, int E>
struct alignas(sizeof(T) * (E & -E)) Part {
    T e[E];
};

template <typename T, int D>
__global__ __launch_bounds__(256) void cache_attend_kernel(Attention a) {
    constexpr int E = D / kWave;
    typedef Part<T, E> P;
    const int lane = threadIdx.x % kWave;
    const long long item = (long long)blockIdx.x * 4 + threadIdx.x / kWave;
    const int t = (int)(item / a.heads), h = (int)(item - (long long)t * a.heads);
    if (t >= a.batch.tokens) return;
    const int b = token_sequence(a.batch, t);
    if (b >= a.batch.batch) return;
    int first, end;
    sequence_rows(a.batch, b, &first, &end);
    if (t < first || t >= end) return;
    const long long len = a.batch.kv_lens[b];
    bool bad = len < 0 || len > a.batch.capacity;
    long long seen = len;
    if (a.causal) seen = len - (a.batch.q_starts[b + 1] - t) + 1;
    const unsigned kvh = h / (a.heads / a.pages.kv_heads), ps = a.pages.page_size.d;
    const P qp = *(const P*)((const T*)a.q + t * a.qs + (long long)h * D + lane * E);
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) q[e] = to_f32(qp.e[e]) * a.scale * kLog2e, o[e] = 0.0f;
    for (int part = 0; part < 2; ++part) {
        const long long n = part ? (bad ? 0 : seen) : a.prefix_len;
        const int* table = part ? a.batch.page_table + (long long)b * a.batch.width : a.prefix_pages;
        for (long long c = 0; c < n; ++c) {
            const unsigned page = a.pages.page_size.div((unsigned)c);
            const int id = table[page];
            if (id < 0 || (unsigned)id >= a.pages.num_pages) {
                bad = true;
                break;
            }
            const size_t row = ((size_t)id * a.pages.kv_heads + kvh) * ps + ((unsigned)c - page * ps);
            const P kp = *(const P*)((const T*)a.pages.k + row * D + lane * E);
            const P vp = *(const P*)((const T*)a.pages.v + row * D + lane * E);
            float s = 0.0f;
            for (int e = 0; e < E; ++e) s += q[e] * to_f32(kp.e[e]);
            s = wave_sum(s);
            const float to = fmaxf(m, s);
            const float keep = m == to ? 1.0f : fast_exp2(m - to), w = fast_exp2(s - to);
            m = to;
            l = l * keep + w;
            for (int e = 0; e < E; ++e) o[e] = o[e] * keep + w * to_f32(vp.e[e]);
        }
    }
    const bool any = a.prefix_len > 0 || seen > 0;
    P out;
    for (int e = 0; e < E; ++e)
        out.e[e] = from_f32<T>(bad ? NAN : any ? o[e] / l : 0.0f);
    *(P*)((T*)a.out + t * a.os + (long long)h * D + lane * E) = out;
}

size_t attention_scratch(const Attention&) { return 0; }

template <typename T>
static void go(const Attention& a, hipStream_t stream) {
    const unsigned grid = (unsigned)(((long long)a.batch.tokens * a.heads + 3) / 4);
    if (a.pages.dim == 64) cache_attend_kernel<T, 64><<<grid, 256, 0, stream>>>(a);
    if (a.pages.dim == 128) cache_attend_kernel<T, 128><<<grid, 256, 0, stream>>>(a);
    if (a.pages.dim == 256) cache_attend_kernel<T, 256><<<grid, 256, 0, stream>>>(a);
    if (a.pages.dim == 768) cache_attend_kernel<T, 768><<<grid, 256, 0, stream>>>(a);
}

bool launch_attention(const Attention& a, void*, hipStream_t stream) {
    if (a.dtype == XATTN_F32) go<float>(a, stream);
    if (a.dtype == XATTN_F16) go<_Float16>(a, stream);
    if (a.dtype == XATTN_BF16) go<__bf16>(a, stream);
    return check_launch("cache_attend_kernel");
}

}  // namespace cache
}  // namespace xattn
