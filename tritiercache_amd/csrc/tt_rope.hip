// tt_rope.hip -- norms of queries and keys for each head, the position rotation
// and the cast to the tiers' type in one pass (gfx950).
//
// A row x of D channels (one head of one token), R = rotary_dim:
//   y = x w / sqrt(mean(x^2) + eps)            (no norm without a weight)
//   z_i       = y_i cos_i - y_(i+R/2) sin_i    i < R/2
//   z_(i+R/2) = y_(i+R/2) cos_(i+R/2) + y_i sin_(i+R/2)
//   z_j       = y_j                            j >= R
// Everything between the load and the store is FP32, and each output value is
// rounded once. Values (the V rows) are only cast.
//
// A row belongs to the D / 16 lanes of a group (a power of two of them, the
// rest idle): a lane holds 8 channels of each half of the rotated part, so
// that both members of a rotated pair sit in one lane, or 16 channels behind
// it, and the norm's sum crosses lanes of one 16-lane row only. Every element
// is read and written once, in 16-byte (float32: two 16-byte) accesses: memory
// is the bound. A prompt of 32k tokens with 32/8 heads of 128 in bfloat16, 805 MB,
// takes 162 us (5.0 TB/s; a copy of 1 GiB reaches 4.76); few tokens take the launch.
#include "tt_wave.h"

#include <algorithm>

namespace tt {
namespace {

typedef __bf16 bf16_t;

// Eight consecutive values as they lie in memory, stored past the caches (cold
// buffers, 32/8 heads of 128, through them and past them: bfloat16 to float32
// at 1777 tokens 19.9 | 16.3 us, at 8192 68.4 | 63.5; float32 to float32 21.7 |
// 20.4, 76.3 | 76.8; bfloat16 to bfloat16 with four heads at 32k 173 | 162). A row starts at a multiple
// of its element's size only: the types say so, and the hardware takes any.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
    typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
    v4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const v4*>(p);
        b = *reinterpret_cast<const v4*>(p + 4);
    }
    __device__ __forceinline__ float get(const int j) const { return j < 4 ? a[j] : b[j - 4]; }
    __device__ __forceinline__ void set(const int j, const float x) {
        if (j < 4)
            a[j] = x;
        else
            b[j - 4] = x;
    }
    __device__ __forceinline__ void store(float* p) const {
        __builtin_nontemporal_store(a, reinterpret_cast<v4*>(p));
        __builtin_nontemporal_store(b, reinterpret_cast<v4*>(p + 4));
    }
};
template <typename T>
struct Eight {
    typedef T v8 __attribute__((ext_vector_type(8), aligned(2)));
    v8 a;
    __device__ __forceinline__ void load(const T* p) { a = *reinterpret_cast<const v8*>(p); }
    __device__ __forceinline__ float get(const int j) const { return static_cast<float>(a[j]); }
    __device__ __forceinline__ void set(const int j, const float x) { a[j] = static_cast<T>(x); }  // to nearest even
    __device__ __forceinline__ void store(T* p) const { __builtin_nontemporal_store(a, reinterpret_cast<v8*>(p)); }
};

template <typename T>
__device__ __forceinline__ void load8_as(const void* p, const int64_t i, float (&x)[8]) {
    Eight<T> e;
    e.load(static_cast<const T*>(p) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = e.get(j);
}
// Eight values of a weight or a table; its type is the launch's.
__device__ __forceinline__ void load8(const void* p, const int64_t i, const int dtype, float (&x)[8]) {
    if (dtype == TT_DTYPE_F32)
        load8_as<float>(p, i, x);
    else if (dtype == TT_DTYPE_F16)
        load8_as<_Float16>(p, i, x);
    else
        load8_as<bf16_t>(p, i, x);
}

// NH: heads of one token that a lane group takes one after another, with the
// token's row of the tables in registers and the loads of all of them in flight.
template <typename In, typename Out, int NH>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const tt_qk_rope a, const int lanes_log2,
                                                           const int chunks_q, const int chunks_kv, const int chunks) {
    const unsigned group = (blockIdx.x * 256u + threadIdx.x) >> lanes_log2;
    const int u = static_cast<int>(threadIdx.x) & ((1 << lanes_log2) - 1);
    const unsigned t = group / static_cast<unsigned>(chunks);
    if (t >= static_cast<unsigned>(a.tokens)) return;
    int c = static_cast<int>(group - t * static_cast<unsigned>(chunks));
    // chunk c: heads of the queries, then of the keys, then of the values
    const int kind = c < chunks_q ? 0 : (c < chunks_q + chunks_kv ? 1 : 2);
    c -= kind == 0 ? 0 : (kind == 1 ? chunks_q : chunks_q + chunks_kv);
    const int heads = kind == 0 ? a.num_q_heads : a.num_kv_heads;
    const int h0 = c * NH;
    const bool on = u < a.head_dim / 16;  // the lane holds channels
    const int half = a.rotary_dim / 2;
    const bool turned = 8 * u < half;
    // the lane's two runs of 8 channels
    const int lo = turned ? 8 * u : a.rotary_dim + 16 * (u - half / 8);
    const int hi = turned ? half + 8 * u : lo + 8;

    const In* src = static_cast<const In*>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v));
    const int64_t ts = kind == 0 ? a.q_token_stride : (kind == 1 ? a.k_token_stride : a.v_token_stride);
    const int64_t hs = kind == 0 ? a.q_head_stride : (kind == 1 ? a.k_head_stride : a.v_head_stride);
    src += static_cast<int64_t>(t) * ts;
    Eight<In> x0[NH] = {}, x1[NH] = {};
#pragma unroll
    for (int i = 0; i < NH; ++i) {
        if (on && h0 + i < heads) {
            x0[i].load(src + (h0 + i) * hs + lo);
            x1[i].load(src + (h0 + i) * hs + hi);
        }
    }
    int64_t row = t;
    if (kind != 0 && a.rows) row = a.rows[t];
    const bool stored = kind == 0 || (row >= 0 && row < a.out_rows);
    float cl[8], ch[8], sl[8], sh[8];
    bool placed = true;  // the token's position has a row in the tables
    if (kind != 2 && a.rotary_dim > 0) {
        const int64_t pos = a.positions ? a.positions[t] : t;
        placed = pos >= 0 && pos < a.table_rows;
        if (turned && placed) {
            load8(a.cos, pos * a.table_stride + lo, a.table_dtype, cl);
            load8(a.cos, pos * a.table_stride + hi, a.table_dtype, ch);
            load8(a.sin, pos * a.table_stride + lo, a.table_dtype, sl);
            load8(a.sin, pos * a.table_stride + hi, a.table_dtype, sh);
        }
    }
    const void* weight = kind == 0 ? a.q_weight : (kind == 1 ? a.k_weight : nullptr);
    float w0[8], w1[8];
    if (weight && on) {
        load8(weight, lo, a.weight_dtype, w0);
        load8(weight, hi, a.weight_dtype, w1);
    }
    Out* dst = static_cast<Out*>(kind == 0 ? a.q_out : (kind == 1 ? a.k_out : a.v_out));
    const int64_t ots = kind == 0 ? a.q_out_token_stride : (kind == 1 ? a.k_out_token_stride : a.v_out_token_stride);
    const int64_t ohs = kind == 0 ? a.q_out_head_stride : (kind == 1 ? a.k_out_head_stride : a.v_out_head_stride);
    dst += row * ots;
#pragma unroll
    for (int i = 0; i < NH; ++i) {
        float y0[8], y1[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y0[j] = x0[i].get(j);
            y1[j] = x1[i].get(j);
        }
        if (weight) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(y0[j], y0[j], __builtin_fmaf(y1[j], y1[j], ss));
            // over the group's lanes, all in one 16-lane row (idle ones hold zeros)
            if (lanes_log2 > 0) ss += dpp<0xB1>(ss);
            if (lanes_log2 > 1) ss += dpp<0x4E>(ss);
            if (lanes_log2 > 2) ss += dpp<0x141>(ss);
            if (lanes_log2 > 3) ss += dpp<0x140>(ss);
            const float r = rsqrtf(ss / static_cast<float>(a.head_dim) + a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y0[j] = y0[j] * r * w0[j];
                y1[j] = y1[j] * r * w1[j];
            }
        }
        Eight<Out> z0, z1;
        if (kind != 2 && turned && placed) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z0.set(j, __builtin_fmaf(y0[j], cl[j], -(y1[j] * sl[j])));
                z1.set(j, __builtin_fmaf(y1[j], ch[j], y0[j] * sh[j]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z0.set(j, placed ? y0[j] : __builtin_nanf(""));
                z1.set(j, placed ? y1[j] : __builtin_nanf(""));
            }
        }
        if (on && stored && h0 + i < heads) {
            z0.store(dst + (h0 + i) * ohs + lo);
            z1.store(dst + (h0 + i) * ohs + hi);
        }
    }
}

template <typename In, typename Out, int NH>
int launch_rope(const tt_qk_rope& a, hipStream_t s, const long long min_blocks, bool* done) {
    int lanes_log2 = 0;
    while ((16 << lanes_log2) < a.head_dim) ++lanes_log2;
    const int cq = (a.num_q_heads + NH - 1) / NH, ckv = (a.num_kv_heads + NH - 1) / NH;
    const int chunks = cq + (a.v ? 2 : 1) * ckv;
    const long long blocks = ((static_cast<long long>(a.tokens) * chunks << lanes_log2) + 255) / 256;
    if (blocks < min_blocks) return TT_OK;
    *done = true;
    if (blocks > 0x00ffffffLL) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "tt_qk_norm_rope: tokens x heads exceed one launch.");
    hipLaunchKernelGGL((qk_norm_rope_kernel<In, Out, NH>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a,
                       lanes_log2, cq, ckv, chunks);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

// Four heads per lane group where that still gives every CU two workgroups, for 16-bit types: of 32/8 heads of 128 in
// bfloat16, one head and four take 191 | 162 us at 32k tokens, 21.7 | 18.6 at 4096, 7.9 | 8.0 at 1000. float32 keeps one
// head: bfloat16 to float32 takes 32.7 | 40.0 us at 4096 tokens, 61.5 | 80.2 at 8192.
template <typename In, typename Out>
int launch_rope(const tt_qk_rope& a, hipStream_t s) {
    bool done = false;
    if constexpr (sizeof(In) == 2 && sizeof(Out) == 2) {
        const int rc = launch_rope<In, Out, 4>(a, s, 512, &done);
        if (done) return rc;
    }
    return launch_rope<In, Out, 1>(a, s, 0, &done);
}

template <typename In>
int launch_rope_out(const tt_qk_rope& a, hipStream_t s) {
    switch (a.out_dtype) {
    case TT_DTYPE_F32: return launch_rope<In, float>(a, s);
    case TT_DTYPE_F16: return launch_rope<In, _Float16>(a, s);
    default: return launch_rope<In, bf16_t>(a, s);
    }
}

bool is_dtype(const int d) { return d == TT_DTYPE_F32 || d == TT_DTYPE_F16 || d == TT_DTYPE_BF16; }

// Whether `rows` x `heads` rows of `d` elements at these strides are apart.
bool apart(const int64_t rows, const int64_t heads, const int64_t ts, const int64_t hs, const int64_t d) {
    if (ts < 0 || hs < 0) return false;
    if (rows <= 1) return heads <= 1 || hs >= d;
    if (heads <= 1) return ts >= d;
    // one of the two strides steps over everything that the other one reaches
    return (hs >= d && ts >= (heads - 1) * hs + d) || (ts >= d && hs >= (rows - 1) * ts + d);
}

int check_rope(const tt_qk_rope& a) {
    if (a.tokens < 0) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "tokens must be non-negative.");
    if (a.num_q_heads <= 0 || a.num_kv_heads <= 0)
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "num_q_heads and num_kv_heads must be positive integers.");
    if (a.head_dim < 16 || a.head_dim > 256 || a.head_dim % 16 != 0)
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "head_dim must be a multiple of 16 of at most 256.");
    if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 16 != 0)
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "rotary_dim must be a multiple of 16 of at most head_dim.");
    if (!is_dtype(a.in_dtype) || !is_dtype(a.out_dtype) || !is_dtype(a.weight_dtype) || !is_dtype(a.table_dtype))
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "in_dtype, out_dtype, weight_dtype and table_dtype must be TT_DTYPE_* values.");
    if (!(a.eps >= 0.0f)) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "eps must be non-negative.");
    if (a.q_token_stride < 0 || a.q_head_stride < 0 || a.k_token_stride < 0 || a.k_head_stride < 0 ||
        a.v_token_stride < 0 || a.v_head_stride < 0)
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "strides must be non-negative.");
    if (a.tokens == 0) return TT_OK;
    if (!a.q || !a.k || !a.q_out || !a.k_out)
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "Argument 'q'/'k'/'q_out'/'k_out' pointer address is NULL.");
    if ((a.v == nullptr) != (a.v_out == nullptr))
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "v and v_out must both be given or both be NULL.");
    if (a.rotary_dim > 0) {
        if (!a.cos || !a.sin) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "Argument 'cos'/'sin' pointer address is NULL.");
        if (a.table_stride < a.rotary_dim)
            TT_FAIL(TT_ERR_INVALID_ARGUMENT, "table_stride must be at least rotary_dim.");
        if (a.table_rows < 0 || (!a.positions && a.table_rows < a.tokens))
            TT_FAIL(TT_ERR_INVALID_ARGUMENT, "without positions the tables need a row for each token.");
    }
    if (a.out_rows < 0 || (!a.rows && a.out_rows < a.tokens))
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "without rows k_out and v_out need a row for each token (out_rows).");
    const int64_t kv_rows = a.rows ? a.out_rows : a.tokens;
    if (!apart(a.tokens, a.num_q_heads, a.q_out_token_stride, a.q_out_head_stride, a.head_dim) ||
        !apart(kv_rows, a.num_kv_heads, a.k_out_token_stride, a.k_out_head_stride, a.head_dim) ||
        (a.v && !apart(kv_rows, a.num_kv_heads, a.v_out_token_stride, a.v_out_head_stride, a.head_dim)))
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "the rows of an output overlap at these strides.");
    // an output in its input's place: only row for row
    auto in_place = [&](const void* x, const void* y, int64_t ts, int64_t hs, int64_t ots, int64_t ohs, bool moved) {
        return x == y && x && (a.in_dtype != a.out_dtype || ts != ots || hs != ohs || moved);
    };
    if (in_place(a.q, a.q_out, a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride, false) ||
        in_place(a.k, a.k_out, a.k_token_stride, a.k_head_stride, a.k_out_token_stride, a.k_out_head_stride, a.rows) ||
        in_place(a.v, a.v_out, a.v_token_stride, a.v_head_stride, a.v_out_token_stride, a.v_out_head_stride, a.rows))
        TT_FAIL(TT_ERR_INVALID_ARGUMENT, "an output in its input's place needs its type and strides, and no rows.");
    return TT_OK;
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_qk_norm_rope(const tt_qk_rope* args, void* stream) {
    clear_error();
    if (!args) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "Argument 'args' pointer address is NULL.");
    const int rc = check_rope(*args);
    if (rc || args->tokens == 0) return rc;
    switch (args->in_dtype) {
    case TT_DTYPE_F32: return launch_rope_out<float>(*args, as_stream(stream));
    case TT_DTYPE_F16: return launch_rope_out<_Float16>(*args, as_stream(stream));
    default: return launch_rope_out<bf16_t>(*args, as_stream(stream));
    }
}
