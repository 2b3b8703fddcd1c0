// Products of a few rows with 4-bit weights: y[m][n] = sum_k x[m][k] w[n][k] + bias[n],
// w[n][k] = scale[n][k / G] * code[n][k] + offset[n][k / G] (no offsets: scale * (code - 8)).  The dense layers of an
// encoder for one query's tokens (MedicalEmbedder.encode of one text, reference src/indexing/embedder.py:65-71), where
// reading the weights is what the layer costs.  gfx950 only.
#include "common.h"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

struct Lin4Args {
    const void* x;
    const uint8_t* codes;
    const void *scales, *offsets, *bias;
    void* y;
    int64_t x_stride, y_stride, m;
    int32_t n, k, group;
};

// One wave per output: lanes over the 32-code pieces of a weight row.
template <typename T>
__global__ __launch_bounds__(256) void linear4_simple_kernel(Lin4Args a) {
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t m = w / a.n;
    const int n = (int)(w - m * a.n);
    if (m >= a.m) return;
    const T* x = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
    const T* scales = reinterpret_cast<const T*>(a.scales) + (int64_t)n * (a.k / a.group);
    const T* offsets = reinterpret_cast<const T*>(a.offsets) + (int64_t)n * (a.k / a.group);
    const uint8_t* codes = a.codes + (int64_t)n * (a.k / 2);
    float sum = 0.f;
    for (int k0 = lane * 32; k0 < a.k; k0 += 64 * 32) {
        const float s = (float)scales[k0 / a.group];
        const float o = a.offsets ? (float)offsets[k0 / a.group] : -8.f * s;
        for (int j = 0; j < 16; ++j) {
            const uint32_t c = codes[(k0 >> 1) + j];
            sum += (s * (float)(c & 15) + o) * (float)x[k0 + 2 * j];
            sum += (s * (float)(c >> 4) + o) * (float)x[k0 + 2 * j + 1];
        }
    }
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) {
        if (a.bias) sum += (float)reinterpret_cast<const T*>(a.bias)[n];
        reinterpret_cast<T*>(a.y)[m * a.y_stride + n] = (T)sum;
    }
}

template <typename T>
int linear4_launch(const Lin4Args& a, hipStream_t stream) {
    const int64_t grid = ceil_div64(a.m * a.n, 4);
    RAG_REQUIRE(grid < (1ll << 31), RAG_ELIMIT, "rag_enc_linear4: too many outputs");
    linear4_simple_kernel<T><<<(unsigned)grid, 256, 0, stream>>>(a);
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

}  // namespace

extern "C" int rag_enc_linear4_dev(const void* d_x, int64_t x_stride, const uint8_t* d_codes, const void* d_scales,
                                   const void* d_offsets, const void* d_bias, int64_t m, int32_t n, int32_t k, int32_t group,
                                   int32_t dtype, void* d_y, int64_t y_stride, void* stream_) {
    const char* me = "rag_enc_linear4";
    RAG_REQUIRE(dtype == RAG_DTYPE_F32 || dtype == RAG_DTYPE_BF16 || dtype == RAG_DTYPE_F16, RAG_EINVAL, "%s: unknown dtype %d", me, dtype);
    RAG_REQUIRE(m >= 0 && n >= 1 && k >= 1, RAG_EINVAL, "%s: bad sizes", me);
    RAG_REQUIRE(group == 32 || group == 64 || group == 128, RAG_ELIMIT, "%s: the group must be 32, 64 or 128 (got %d)", me, group);
    RAG_REQUIRE(k % group == 0, RAG_ELIMIT, "%s: k = %d is not a multiple of the group %d", me, k, group);
    RAG_REQUIRE(m < (1ll << 31) && n < (1 << 30) && k < (1 << 30), RAG_ELIMIT, "%s: sizes beyond the limit", me);
    if (m == 0) return RAG_OK;
    RAG_REQUIRE(d_x && d_codes && d_scales && d_y, RAG_EINVAL, "%s: null pointer", me);
    const int size = dtype == RAG_DTYPE_F32 ? 4 : 2;
    RAG_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && reinterpret_cast<uintptr_t>(d_codes) % 16 == 0 && x_stride * size % 16 == 0,
                RAG_EINVAL, "%s: x, its rows and the codes must be 16-byte aligned", me);
    RAG_REQUIRE(reinterpret_cast<uintptr_t>(d_scales) % size == 0 && reinterpret_cast<uintptr_t>(d_offsets) % size == 0 &&
                reinterpret_cast<uintptr_t>(d_bias) % size == 0 && reinterpret_cast<uintptr_t>(d_y) % size == 0, RAG_EINVAL,
                "%s: misaligned pointer", me);
    RAG_REQUIRE((m == 1 || x_stride >= k) && (m == 1 || y_stride >= n), RAG_EINVAL, "%s: a row's stride is smaller than the row", me);
    Lin4Args a{d_x, d_codes, d_scales, d_offsets, d_bias, d_y, x_stride, y_stride, m, n, k, group};
    hipStream_t stream = (hipStream_t)stream_;
    if (dtype == RAG_DTYPE_F32) return linear4_launch<float>(a, stream);
    if (dtype == RAG_DTYPE_BF16) return linear4_launch<bf16>(a, stream);
    return linear4_launch<f16>(a, stream);
}
