// Attention with a sliding window and a few first tokens that stay visible, over packed sequences whose keys may be
// kept from earlier calls: self-attention of long documents in local layers, and the few new tokens of a query behind a
// kept prefix.  For encoders with windowed layers behind MedicalEmbedder.encode (reference
// src/indexing/embedder.py:65-71).  gfx950 only.
//
// Query j of a sequence with nq queries and nk keys stands at position p = nk - nq + j.  It sees key c (0 <= c < nk) if
//   c - p <= right (right < 0: no limit)   and   (p - c <= left (left < 0: no limit)  or  c < n_sinks)
// that is, the keys [0, s) and [lo, hi) of Seen below.  out = sum softmax(scale q.k) v over them; none: 0.
#include "common.h"

#include <math.h>

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T, int N> struct Vec { typedef T type __attribute__((ext_vector_type(N))); };

struct WinArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t* cu_q;
    const int64_t* k_start;          // NULL: the keys of a sequence are the rows of its queries
    const int32_t* k_len;
    int64_t q_stride, k_row, k_head, v_row, v_head, out_stride;
    int64_t total_q, total_k;
    int32_t n_seq, max_q, max_k, hq, hkv, left, right, sinks;
    float scale;                     // scale * log2(e): the softmax is taken to base 2
};

struct Seq { int64_t q0, k0; int nq, nk; };

// The sequence's rows, checked against the arrays.  False (and flagged): not a sequence of this batch.
__device__ __forceinline__ bool load_seq(const WinArgs& a, int i, Seq& s, uint32_t* fault) {
    s.q0 = a.cu_q[i];
    const int64_t nq = (int64_t)a.cu_q[i + 1] - s.q0;
    int64_t nk = nq;
    s.k0 = s.q0;
    if (a.k_start != nullptr) { s.k0 = a.k_start[i]; nk = a.k_len[i]; }
    const bool q_ok = s.q0 >= 0 && nq >= 0 && nq <= a.max_q && s.q0 <= a.total_q - nq;
    const bool k_ok = s.k0 >= 0 && nk >= 0 && nk <= a.max_k && s.k0 <= a.total_k - nk;
    s.nq = (int)nq;
    s.nk = (int)nk;
    if (!(q_ok && k_ok) && threadIdx.x == 0) rag_flag(fault, q_ok ? RAG_FAULT_KV_ROW : RAG_FAULT_SEGMENT);
    return q_ok && k_ok;
}

struct Seen { int s, lo, hi; };      // visible keys: [0, s) and [lo, hi), s <= lo <= hi

__device__ __forceinline__ Seen seen_by(const WinArgs& a, int p, int nk) {
    Seen w;
    w.hi = a.right < 0 ? nk : max(0, min(nk, p + a.right + 1));
    w.lo = a.left < 0 ? 0 : min(w.hi, max(0, p - a.left));
    w.s = min(a.sinks, w.lo);
    return w;
}

// One wave, one query row of one head.  Reads no key and no value that the query does not see.
template <typename T, int D>
__device__ void attend_row(const WinArgs& a, const Seq& sq, int j, int head, int lane) {
    typedef typename Vec<T, 8>::type v8;
    constexpr int DL = D / 2;                                // a lane owns 2 dimensions of the result ...
    constexpr int PARTS = 64 / DL;                           // ... of one of these shares of the keys
    const int kvh = head / (a.hq / a.hkv);
    const T* q = reinterpret_cast<const T*>(a.q) + (sq.q0 + j) * a.q_stride + (int64_t)head * D;
    const T* k = reinterpret_cast<const T*>(a.k) + sq.k0 * a.k_row + (int64_t)kvh * a.k_head;
    const T* v = reinterpret_cast<const T*>(a.v) + sq.k0 * a.v_row + (int64_t)kvh * a.v_head;
    const Seen w = seen_by(a, sq.nk - sq.nq + j, sq.nk);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    const int total = w.s + (w.hi - w.lo);
    const int d0 = 2 * (lane % DL), part = lane / DL;
    for (int base = 0; base < total; base += 64) {
        const int n = min(64, total - base);
        float s = -INFINITY;
        if (lane < n) {
            const int key = base + lane < w.s ? base + lane : base + lane - w.s + w.lo;
            const T* kr = k + (int64_t)key * a.k_row;
            float dot = 0.f;
            for (int d = 0; d < D; d += 8) {
                const v8 kv = *reinterpret_cast<const v8*>(kr + d), qv = *reinterpret_cast<const v8*>(q + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = fmaf((float)kv[e], (float)qv[e], dot);
            }
            s = dot * a.scale;
        }
        float mx = s;
        bool bad = s != s;                                   // fmaxf would drop a NaN
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        const float m_new = fmaxf(m, mx);
        const float top = m_new == -INFINITY ? 0.f : m_new;
        const float p = exp2f(s - top);
        float sum = lane < n ? p : 0.f;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
        (void)bad;
        const float alpha = exp2f(m - top);
        l = l * alpha + sum;
        o0 *= alpha;
        o1 *= alpha;
        m = m_new;
        for (int i = 0; i < n; i += PARTS) {
            const int mine = i + part;
            const float pi = __shfl(p, min(mine, 63), 64);
            if (mine < n) {
                const int key = base + mine < w.s ? base + mine : base + mine - w.s + w.lo;
                const T* vr = v + (int64_t)key * a.v_row + d0;
                o0 = fmaf(pi, (float)vr[0], o0);
                o1 = fmaf(pi, (float)vr[1], o1);
            }
        }
    }
#pragma unroll
    for (int o = DL; o < 64; o <<= 1) { o0 += __shfl_xor(o0, o, 64); o1 += __shfl_xor(o1, o, 64); }
    if (part == 0) {
        T* dst = reinterpret_cast<T*>(a.out) + (sq.q0 + j) * a.out_stride + (int64_t)head * D + d0;
        const float inv = total > 0 ? 1.f / l : 0.f;
        dst[0] = (T)(total > 0 ? o0 * inv : 0.f);
        dst[1] = (T)(total > 0 ? o1 * inv : 0.f);
    }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void window_row_kernel(WinArgs a, uint32_t* fault) {
    const int rows4 = (a.max_q + 3) / 4;
    const int seq = (int)(blockIdx.x / rows4);
    const int j = (int)(blockIdx.x % rows4) * 4 + (int)(threadIdx.x >> 6);
    const int head = (int)blockIdx.y;
    Seq s;
    if (!load_seq(a, seq, s, fault) || j >= s.nq) return;
    attend_row<T, D>(a, s, j, head, threadIdx.x & 63);
}

template <typename T, int D>
int window_launch(const WinArgs& a, hipStream_t stream) {
    const int64_t grid = (int64_t)a.n_seq * ((a.max_q + 3) / 4);
    RAG_REQUIRE(grid < (1ll << 31), RAG_ELIMIT, "rag_enc_attention_window: too many query rows");
    window_row_kernel<T, D><<<dim3((unsigned)grid, (unsigned)a.hq), 256, 0, stream>>>(a, rag_fault_word());
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

template <typename T>
int window_by_dim(const WinArgs& a, int D, hipStream_t stream) {
    if (D == 32) return window_launch<T, 32>(a, stream);
    if (D == 64) return window_launch<T, 64>(a, stream);
    return window_launch<T, 128>(a, stream);
}

}  // namespace

extern "C" int64_t rag_enc_attention_window_workspace(int64_t total_q, int32_t n_seq, int32_t max_q_len, int32_t max_k_len,
                                                      int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                      int32_t window_left, int32_t window_right, int32_t n_sinks) {
    (void)total_q; (void)n_seq; (void)max_q_len; (void)max_k_len; (void)n_q_heads; (void)n_kv_heads; (void)head_dim;
    (void)window_left; (void)window_right; (void)n_sinks;
    return 0;
}

extern "C" int rag_enc_attention_window_dev(const void* d_q, int64_t q_stride, const void* d_k, int64_t k_row_stride,
                                            int64_t k_head_stride, const void* d_v, int64_t v_row_stride, int64_t v_head_stride,
                                            const int32_t* d_cu_q, int64_t total_q, const int64_t* d_k_start,
                                            const int32_t* d_k_len, int64_t total_k, int32_t n_seq, int32_t max_q_len,
                                            int32_t max_k_len, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                                            int32_t window_left, int32_t window_right, int32_t n_sinks, int32_t dtype, void* d_out,
                                            int64_t out_stride, void* d_workspace, int64_t workspace_bytes, void* stream_) {
    const char* me = "rag_enc_attention_window";
    RAG_REQUIRE(dtype == RAG_DTYPE_F32 || dtype == RAG_DTYPE_BF16 || dtype == RAG_DTYPE_F16, RAG_EINVAL, "%s: unknown dtype %d", me, dtype);
    RAG_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, RAG_ELIMIT, "%s: head_dim must be 32, 64 or 128 (got %d)", me, head_dim);
    RAG_REQUIRE(n_seq >= 0 && max_q_len >= 0 && max_k_len >= 0 && total_q >= 0 && total_k >= 0, RAG_EINVAL, "%s: bad sizes", me);
    RAG_REQUIRE(total_q < (1ll << 31) && max_q_len < (1 << 30) && max_k_len < (1 << 30), RAG_ELIMIT, "%s: sizes beyond the limit", me);
    RAG_REQUIRE(n_kv_heads >= 1 && n_q_heads >= 1 && n_q_heads <= 4096 && n_q_heads % n_kv_heads == 0, RAG_EINVAL,
                "%s: the query heads must be a multiple of the key/value heads", me);
    RAG_REQUIRE(window_left >= -1 && window_right >= -1 && n_sinks >= 0, RAG_EINVAL, "%s: bad window", me);
    RAG_REQUIRE(isfinite(scale), RAG_EINVAL, "%s: bad scale", me);
    RAG_REQUIRE((d_k_start == nullptr) == (d_k_len == nullptr), RAG_EINVAL, "%s: key starts and key lengths come together", me);
    if (n_seq == 0 || total_q == 0 || max_q_len == 0) return RAG_OK;
    RAG_REQUIRE(d_q && d_cu_q && d_out && ((d_k && d_v) || total_k == 0), RAG_EINVAL, "%s: null pointer", me);
    const int size = dtype == RAG_DTYPE_F32 ? 4 : 2;
    const auto off = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; };
    RAG_REQUIRE(!off(d_q) && !off(d_k) && !off(d_v) && !off(d_out), RAG_EINVAL, "%s: pointers must be 16-byte aligned", me);
    RAG_REQUIRE(q_stride * size % 16 == 0 && k_row_stride * size % 16 == 0 && k_head_stride * size % 16 == 0 && v_row_stride * size % 16 == 0 &&
                v_head_stride * size % 16 == 0 && out_stride * size % 16 == 0, RAG_EINVAL, "%s: strides must be multiples of 16 bytes", me);
    RAG_REQUIRE(q_stride >= (int64_t)n_q_heads * head_dim && out_stride >= (int64_t)n_q_heads * head_dim, RAG_EINVAL,
                "%s: a row's stride is smaller than the row", me);
    RAG_REQUIRE(workspace_bytes >= 0, RAG_EINVAL, "%s: bad workspace", me);
    WinArgs a;
    a.q = d_q; a.k = d_k; a.v = d_v; a.out = d_out; a.cu_q = d_cu_q; a.k_start = d_k_start; a.k_len = d_k_len;
    a.q_stride = q_stride; a.k_row = k_row_stride; a.k_head = k_head_stride; a.v_row = v_row_stride; a.v_head = v_head_stride;
    a.out_stride = out_stride; a.total_q = total_q; a.total_k = total_k;
    a.n_seq = n_seq; a.max_q = max_q_len; a.max_k = d_k_start ? max_k_len : max_q_len; a.hq = n_q_heads; a.hkv = n_kv_heads;
    const int far = 1 << 30;                                 // beyond every length: no limit, and no overflow
    a.left = window_left >= far ? -1 : window_left;
    a.right = window_right >= far ? -1 : window_right;
    a.sinks = n_sinks;
    a.scale = scale * 1.4426950408889634f;
    (void)d_workspace;
    hipStream_t stream = (hipStream_t)stream_;
    if (dtype == RAG_DTYPE_F32) return window_by_dim<float>(a, head_dim, stream);
    if (dtype == RAG_DTYPE_BF16) return window_by_dim<bf16>(a, head_dim, stream);
    return window_by_dim<f16>(a, head_dim, stream);
}
