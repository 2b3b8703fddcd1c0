// Norms of queries and keys for each head and the rotation by position, in one pass over the q|k|v projection's output,
// with keys and values written where the attention reads them.  For encoders with rotary positions,
// beside the BERT encoders of MedicalEmbedder (reference src/indexing/embedder.py:65-71), which have none.  gfx950 only.
//
//   n = x * gamma / sqrt(mean(x^2) + eps)        (gamma NULL: n = x)
//   (n_a, n_b) -> (n_a cos - n_b sin, n_b cos + n_a sin),  angle = pos * inv_freq[i],
//   (a, b) = (i, i + R/2) or (2i, 2i + 1), i < R/2; dimensions from R on are not rotated
//
// Bytes bound: an element is read once, written once, and costs about fifteen instructions.  A head is D/8 lanes of a
// wave; a lane owns two pieces of four dimensions which are rotated against each other, so the rotation needs no
// exchange between lanes and the sum of squares only the D/8 lanes of the head.  Angles are the same for every head of
// a token: a lane computes one, takes its four from the others and uses them for all heads of the wave (four computed
// by every lane: 16384 tokens 73 us for 69, 24 heads of 32 17.9 for 15.5).  They are reduced to a fraction of
// a turn in 64 bits (a 32-bit product is off by 2^-24 of the angle itself, 0.002 radians at position 32768) and only
// the sine and cosine of the remainder are taken in 32 bits, so there is no table to read or to size.
// Measured: 16384 tokens of 32 query and 8 key heads of 128, bf16, 69 us, 4.86 TB/s (a large copy moves 4.7); 65536 tokens
// of 16 and 8 heads of 128, half of each rotated, f16, 156 us, 5.2 TB/s; one token 2.5 us, of which an empty launch is 1.6.
#include "common.h"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> struct Vec4;
template <> struct Vec4<bf16> { typedef bf16 type __attribute__((ext_vector_type(4))); };
template <> struct Vec4<f16> { typedef f16 type __attribute__((ext_vector_type(4))); };
template <> struct Vec4<float> { typedef float type __attribute__((ext_vector_type(4))); };

struct RopeArgs {
    const void* qkv;
    const int32_t* pos;
    const void *gamma_q, *gamma_k;
    const double* inv_freq;
    void *q_out, *k_out, *v_out;
    const int64_t* kv_row;
    int64_t stride, q_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride;
    int64_t n_tokens, n_rows;
    int32_t rot, hq, hkv, heads;      // heads: hq + hkv, and another hkv where values are copied
    int32_t chunks;                   // waves per token
    float eps;
};

constexpr int ROPE_NT = 256;

// U: heads a lane takes, all their loads issued before the first is used
template <typename T, int D, bool INTER, int U>
__global__ __launch_bounds__(ROPE_NT) void qk_norm_rope_kernel(RopeArgs a, uint32_t* fault) {
    typedef typename Vec4<T>::type v4;
    constexpr int L = D / 8;          // lanes of a head
    constexpr int HPW = 64 / L;       // heads of a wave at a time
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * (ROPE_NT / 64) + (threadIdx.x >> 6);
    const int64_t t = w / a.chunks;
    const int chunk = (int)(w - t * a.chunks);
    if (t >= a.n_tokens) return;
    const int p = lane % L;
    const bool turns = 8 * p < a.rot;
    const int off_a = INTER || !turns ? 8 * p : 4 * p;
    const int off_b = INTER || !turns ? 8 * p + 4 : 4 * p + a.rot / 2;

    const T* row = reinterpret_cast<const T*>(a.qkv) + t * a.stride;
    v4 xa[U], xb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = (chunk * U + u) * HPW + lane / L;
        if (head < a.heads) {
            xa[u] = *reinterpret_cast<const v4*>(row + (int64_t)head * D + off_a);
            xb[u] = *reinterpret_cast<const v4*>(row + (int64_t)head * D + off_b);
        }
    }
    const int64_t kv = a.kv_row != nullptr ? a.kv_row[t] : t;
    const bool kv_ok = kv >= 0 && kv < a.n_rows;
    if (kv >= a.n_rows && chunk == 0 && lane == 0) rag_flag(fault, RAG_FAULT_KV_ROW);

    // an angle a lane (at most 64), then the lane's four from those; beyond rot / 2: no turn
    float my_co = 1.f, my_si = 0.f;
    if (lane < a.rot / 2) {
        const double turn = (double)a.pos[t] * 0.15915494309189533577 * a.inv_freq[lane];          // 1 / (2 pi)
        sincospif(2.f * (float)(turn - rint(turn)), &my_si, &my_co);
    }
    float co[4], si[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        co[j] = __shfl(my_co, 4 * p + j, 64);
        si[j] = __shfl(my_si, 4 * p + j, 64);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = (chunk * U + u) * HPW + lane / L;
        if (head >= a.heads) continue;                       // (the lanes of a head stay together)
        const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
        T* dst;
        if (is_q) {
            dst = reinterpret_cast<T*>(a.q_out) + t * a.q_stride + (int64_t)head * D;
        } else if (!is_v) {
            dst = reinterpret_cast<T*>(a.k_out) + kv * a.k_row_stride + (int64_t)(head - a.hq) * a.k_head_stride;
        } else {
            dst = reinterpret_cast<T*>(a.v_out) + kv * a.v_row_stride + (int64_t)(head - a.hq - a.hkv) * a.v_head_stride;
        }
        if (is_v) {
            if (kv_ok) {
                *reinterpret_cast<v4*>(dst + off_a) = xa[u];
                *reinterpret_cast<v4*>(dst + off_b) = xb[u];
            }
            continue;
        }
        float fa[4], fb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) { fa[j] = (float)xa[u][j]; fb[j] = (float)xb[u][j]; }
        const T* gamma = reinterpret_cast<const T*>(is_q ? a.gamma_q : a.gamma_k);
        if (gamma != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) ss += fa[j] * fa[j] + fb[j] * fb[j];
#pragma unroll
            for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o, 64);
            const float inv = 1.f / sqrtf(ss * (1.f / D) + a.eps);
            const v4 ga = *reinterpret_cast<const v4*>(gamma + off_a), gb = *reinterpret_cast<const v4*>(gamma + off_b);
#pragma unroll
            for (int j = 0; j < 4; ++j) { fa[j] *= inv * (float)ga[j]; fb[j] *= inv * (float)gb[j]; }
        }
        // Dimensions behind rot_dim stay as they are: a product with a sine of 0 would pass an infinity or a NaN on.
        if (turns) {
            float ra[4], rb[4];
            if (INTER) {                                      // pairs (0, 1), (2, 3) of each piece
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    ra[2 * j] = fa[2 * j] * co[j] - fa[2 * j + 1] * si[j];
                    ra[2 * j + 1] = fa[2 * j + 1] * co[j] + fa[2 * j] * si[j];
                    rb[2 * j] = fb[2 * j] * co[2 + j] - fb[2 * j + 1] * si[2 + j];
                    rb[2 * j + 1] = fb[2 * j + 1] * co[2 + j] + fb[2 * j] * si[2 + j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ra[j] = fa[j] * co[j] - fb[j] * si[j];
                    rb[j] = fb[j] * co[j] + fa[j] * si[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { fa[j] = ra[j]; fb[j] = rb[j]; }
        }
        v4 ya, yb;
#pragma unroll
        for (int j = 0; j < 4; ++j) { ya[j] = (T)fa[j]; yb[j] = (T)fb[j]; }
        if (is_q || kv_ok) {
            *reinterpret_cast<v4*>(dst + off_a) = ya;
            *reinterpret_cast<v4*>(dst + off_b) = yb;
        }
    }
}

template <typename T, int D, int U>
int rope_launch(RopeArgs a, bool inter, hipStream_t stream) {
    const int per_wave = 64 / (D / 8) * U;
    a.chunks = (a.heads + per_wave - 1) / per_wave;
    const int64_t grid = ceil_div64(a.n_tokens * a.chunks, ROPE_NT / 64);
    RAG_REQUIRE(grid < (1ll << 24), RAG_ELIMIT, "rag_enc_qk_norm_rope: too many tokens");
    if (inter) qk_norm_rope_kernel<T, D, true, U><<<(unsigned)grid, ROPE_NT, 0, stream>>>(a, rag_fault_word());
    else qk_norm_rope_kernel<T, D, false, U><<<(unsigned)grid, ROPE_NT, 0, stream>>>(a, rag_fault_word());
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

// One head a lane while the waves are on the chip at once, 32 a compute unit: less to do one after the other (16 + 8 heads
// of 128, bf16: one token 2.6 us, with four heads 4.2, 512 tokens 3.5 and 5.1, 1024 5.2 and 5.7).  Beyond that four: more bytes in
// flight and the angles for four heads at once (2048 tokens 7.8 us, with one head 8.2, 8192 22.5 and 25.2).
template <typename T, int D>
int rope_by_size(const RopeArgs& a, bool inter, hipStream_t stream) {
    const int64_t waves = a.n_tokens * ((a.heads + 512 / D - 1) / (512 / D));
    return waves <= 8192 ? rope_launch<T, D, 1>(a, inter, stream) : rope_launch<T, D, 4>(a, inter, stream);
}

template <typename T>
int rope_by_dim(const RopeArgs& a, int D, bool inter, hipStream_t stream) {
    if (D == 32) return rope_by_size<T, 32>(a, inter, stream);
    if (D == 64) return rope_by_size<T, 64>(a, inter, stream);
    return rope_by_size<T, 128>(a, inter, stream);
}

}  // namespace

extern "C" int rag_enc_qk_norm_rope_dev(const void* d_qkv, int64_t qkv_stride, const int32_t* d_pos, const void* d_gamma_q,
                                        const void* d_gamma_k, float eps, const double* d_inv_freq, int32_t rot_dim,
                                        int32_t interleaved, int64_t n_tokens, int32_t n_q_heads, int32_t n_kv_heads,
                                        int32_t head_dim, int32_t dtype, void* d_q_out, int64_t q_stride, void* d_k_out,
                                        int64_t k_row_stride, int64_t k_head_stride, void* d_v_out, int64_t v_row_stride,
                                        int64_t v_head_stride, const int64_t* d_kv_row, int64_t n_kv_rows, void* stream_) {
    const char* me = "rag_enc_qk_norm_rope";
    RAG_REQUIRE(dtype == RAG_DTYPE_F32 || dtype == RAG_DTYPE_BF16 || dtype == RAG_DTYPE_F16, RAG_EINVAL, "%s: unknown dtype %d", me, dtype);
    RAG_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, RAG_ELIMIT, "%s: head_dim must be 32, 64 or 128 (got %d)", me, head_dim);
    RAG_REQUIRE(n_tokens >= 0 && n_q_heads >= 1 && n_kv_heads >= 1 && n_q_heads <= 4096 && n_kv_heads <= 4096, RAG_EINVAL,
                "%s: bad token or head count", me);
    RAG_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 8 == 0, RAG_ELIMIT,
                "%s: rot_dim must be a multiple of 8 up to the head size (got %d)", me, rot_dim);
    RAG_REQUIRE(n_kv_rows >= 0 && (d_kv_row != nullptr || n_kv_rows >= n_tokens), RAG_EINVAL, "%s: fewer key/value rows than tokens", me);
    if (n_tokens == 0) return RAG_OK;
    RAG_REQUIRE(d_qkv && d_q_out && d_k_out && (rot_dim == 0 || (d_pos && d_inv_freq)), RAG_EINVAL, "%s: null pointer", me);
    const int size = dtype == RAG_DTYPE_F32 ? 4 : 2;
    const int64_t vec = 4 * size;                            // bytes of a piece
    const auto off = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)vec; };
    RAG_REQUIRE(!off(d_qkv) && !off(d_gamma_q) && !off(d_gamma_k) && !off(d_q_out) && !off(d_k_out) && !off(d_v_out), RAG_EINVAL,
                "%s: pointers must be %d-byte aligned", me, (int)vec);
    RAG_REQUIRE(qkv_stride % 4 == 0 && q_stride % 4 == 0 && k_row_stride % 4 == 0 && k_head_stride % 4 == 0 && v_row_stride % 4 == 0 &&
                v_head_stride % 4 == 0, RAG_EINVAL, "%s: strides must be multiples of 4 elements", me);
    RAG_REQUIRE(qkv_stride >= (int64_t)(n_q_heads + 2 * n_kv_heads) * head_dim && q_stride >= (int64_t)n_q_heads * head_dim, RAG_EINVAL,
                "%s: a row's stride is smaller than the row", me);
    // (rows of every head may lie together, [head][row], so a stride may be smaller than a row of all heads, but not than a head)
    const auto apart = [&](int64_t stride, int64_t n) { return n <= 1 || stride >= head_dim || stride <= -head_dim; };
    RAG_REQUIRE(apart(k_row_stride, n_kv_rows) && apart(k_head_stride, n_kv_heads) &&
                (!d_v_out || (apart(v_row_stride, n_kv_rows) && apart(v_head_stride, n_kv_heads))), RAG_EINVAL,
                "%s: rows or heads of the keys or values overlap", me);
    RopeArgs a;
    a.qkv = d_qkv; a.pos = d_pos; a.gamma_q = d_gamma_q; a.gamma_k = d_gamma_k; a.inv_freq = d_inv_freq;
    a.q_out = d_q_out; a.k_out = d_k_out; a.v_out = d_v_out; a.kv_row = d_kv_row;
    a.stride = qkv_stride; a.q_stride = q_stride; a.k_row_stride = k_row_stride; a.k_head_stride = k_head_stride;
    a.v_row_stride = v_row_stride; a.v_head_stride = v_head_stride;
    a.n_tokens = n_tokens; a.n_rows = n_kv_rows;
    a.rot = rot_dim; a.hq = n_q_heads; a.hkv = n_kv_heads; a.heads = n_q_heads + (d_v_out ? 2 : 1) * n_kv_heads;
    a.eps = eps;
    RAG_REQUIRE(n_tokens < (1ll << 40), RAG_ELIMIT, "%s: too many tokens", me);
    hipStream_t stream = (hipStream_t)stream_;
    if (dtype == RAG_DTYPE_F32) return rope_by_dim<float>(a, head_dim, interleaved != 0, stream);
    if (dtype == RAG_DTYPE_BF16) return rope_by_dim<bf16>(a, head_dim, interleaved != 0, stream);
    return rope_by_dim<f16>(a, head_dim, interleaved != 0, stream);
}
