// tt_shared.hip -- decode attention of a batch whose sequences share a prefix (gfx950).
//
// The queries of all sequences that read one KV head form one matrix, so the
// prefix's keys and values are unpacked once and multiplied on the matrix
// cores with many rows, instead of once per sequence. For a KV head, with rows
// r = (sequence, query head of the group), tokens t, channels c:
//   S = Q K^T (log2 units), P = 2^(S - m), l = P 1, O = P V
// over a share of the tokens gives one (m, l, O) partial per row; the merge of
// the ragged batch joins them with the partials of each sequence's own tiers.
//
// The matrix instructions multiply f16, the operator is FP32: every operand is
// a high and a low f16 part (x = hi + lo to about 21 bits) and a product is
// hi hi + hi lo + lo hi, summed in FP32.
// f16 covers 2^-14 .. 2^16 with all its bits, so the parts are scaled by
// powers of two: Q by its row's largest value (to below 2^12), K and V by the
// first tile's (k_exp, v_exp: to 2^11 .. 2^12; a tile with larger values than
// the limit is staged again with another exponent), P by the running reference
// m = max - 5 (P <= 2^14 with the slack of the lazy rescale). The codes of
// packed V are exact in one part, and their scales go into P.
//
// Bounds, for 64 sequences behind 32k tokens with 32/8 heads of 128: the
// products, 34 GFLOP, are 86 with the parts (75 us at the 1149 TFLOP/s that a
// large f16 product reaches on this card), the prefix's bytes 50 MB (11 us). The
// prefix takes 106 us: 40% of the cycles are matrix instructions' (at about 2.0
// GHz), about as many the VALU's, which unpacks, exponentiates and splits P
// (some 330 instructions per wave and tile of 32 tokens x 32 rows against 40
// matrix ones), and the two hardly overlap with two waves per SIMD, the most
// that 250 registers allow. Measured without gain: the two halves of the waves
// half a tile apart, K and V staged by different waves, priorities of the waves,
// operands read two steps ahead.
#include "tt_shared.h"
#include "tt_wave.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tt {
namespace {

// Rows of a KV head that a wave can take alone, and the tiles per CU (of all heads) from which on each wave takes tiles of its
// own, four or more (whole call, a group's tiles | a wave's: 8 sequences, 32/32 heads of 80 behind 4k 37.1 | 29.8 us, behind
// 16k 86.0 | 55.6, behind 2k 29.0 | 30.7; 32/32 heads of 128 behind 4k 43.1 | 38.4; 32/8 behind 8k 39.4 | 40.8, behind 16k
// 46.6 | 46.0, behind 64k 92 | 76; slots of two tiles cost 12/4 heads of 96 behind 16k 40.5 instead of 34.2).
constexpr int kLoneRows = 32;
constexpr int kLoneTiles = 12;
constexpr double kDenseCost = 1.5;  // an FP32 tile in packed ones

// What the two ways to attend to a prefix take, in us, to choose between them. Multiplied for all sequences, a fixed part
// that grows with head_dim (kSharedUs + head_dim / 16), its tiles and its merge; ...
constexpr double kSharedUs = 14.0;
constexpr double kMergeRate = 4.5e6;  // bytes per us of partials, written and read
double tile_us(const int D) { return 2.0 + D / 256.0; }
// ... read once per sequence, by matrix products (head_dim 128) or the VALU, the launch and the tokens. Fitted to 1 to 32
// sequences behind 512 to 16k tokens with seven head shapes: the choice is the faster one or within 12% of it in 246 of
// 252 of them, and 28% slower at worst. (Whole call, multiplied against read by each, 32/8 heads of 128: 8 sequences
// behind 4k 34.6 | 27.6 us, 16 behind 2k 32.0 | 27.5, 16 behind 8k 43.2 | 50.7, 32 behind 2k 37.0 | 48.4; heads of 64: 4
// behind 8k 25.6 | 24.7, 16 behind 4k 26.6 | 42.9.)
double walk_us(const int nseq, const double tokens, const int Hq, const int Hkv, const int D) {
    if (D == 128) return 11.0 + nseq * Hkv * (0.045 + 0.34e-6 * tokens * D);
    return 11.0 + 1e-6 * nseq * tokens * D * (0.2 * Hkv + 0.17 * Hq);
}

constexpr int kWideDC = 8;          // 32-channel chunks of a head in the kernel for head dims above 128
constexpr int kTile = 32;           // tokens of a tile: FP32 rows or packed slots
constexpr float kLimit = 65000.0f;  // scaled keys and values stay below this
// log2 of P's largest value when a row's reference moves, and how much further
// its logits may rise before it moves again: P <= 2^14. (With 12 and 2 a wave of
// 32 rows rescaled in every other tile.)
constexpr float kUp = 5.0f;
constexpr float kSlack = 9.0f;

// LDS of one tile: K as [token][channel], V as [channel][token in MFMA order],
// high and low parts (V's packed codes: one part), and of packed tiles V's
// scale and zero by token. The row strides put the 16-byte reads of eight
// lanes and the 8-byte writes of sixteen in distinct banks.
template <int DC>
struct TileLds {
    static constexpr int KS = 64 * DC + 16;           // bytes per K row
    static constexpr int VS = 80;                     // bytes per V row
    static constexpr int KHI = 0;
    static constexpr int KLO = KHI + kTile * KS;
    static constexpr int V = KLO + kTile * KS;
    static constexpr int VLO = V + 32 * DC * VS;
    static constexpr int VMETA = VLO + 32 * DC * VS;  // [scale | zero][32] f32
    static constexpr int BYTES = VMETA + 2 * kTile * 4;
};

constexpr int kLds = 160 * 1024;  // of a CU

// Workgroups of WM waves, all on the same tile with rows of their own: two
// tiles in LDS in turn, two waves per SIMD.
template <int DC, int WM>
struct Config {
    static constexpr int ROWS = (DC > 4 ? 16 : 32) * WM;
    static constexpr int LDS = 2 * TileLds<DC>::BYTES + 16;
    static constexpr int PER_CU = kLds / LDS < 8 / WM ? kLds / LDS : 8 / WM;
    static constexpr int PER_EU = PER_CU * WM >= 8 ? 2 : 1;
};

struct SharedArgs {
    const tt_decode_seq* __restrict__ seqs;
    tt_decode_seq prefix;
    float* ml;
    float* acc;
    float scale2;         // log2(e) / sqrt(head_dim)
    int nseq, Hq, Hkv, D, kgs, meta_fp16;
    int prefix_slots;     // of which the first packed_slots share the packed tiles
    int packed_slots;
    int chunks;           // row chunks per KV head
    int slot_base[kMaxBatchSeqs + 1];
};

// (hi, lo) of two values, both rounded to nearest: hi + lo is x to 23 bits, off to either side (truncated parts would make
// every product too small, and the prefix's weights with it). `neg1` is -1 whose value the compiler does not know: the
// remainder is then one mixed fused multiply-add instead of a conversion and a subtraction.
__device__ __forceinline__ uint2 parts(const float x0, const float x1, const float neg1) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const mf_h2 hi = __builtin_convertvector((f2{x0, x1}), mf_h2);
    const float r0 = __builtin_fmaf(static_cast<float>(hi.x), neg1, x0), r1 = __builtin_fmaf(static_cast<float>(hi.y), neg1, x1);
    const mf_h2 lo = __builtin_convertvector((f2{r0, r1}), mf_h2);
    return make_uint2(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo));
}

// The exponent of the scale for keys and values up to `peak` (0: not known): 16 peak 2^-e in 2^11 .. 2^12 for `below` = 8, which
// leaves a factor of 16 for the tiles to come.
__device__ __forceinline__ int exponent(const float peak, const int below) {
    return peak > 0.0f ? max(scalar(__builtin_amdgcn_frexp_expf(fminf(peak, 3.0e38f))) - below, -118) : 0;
}

// The largest x (>= 0) of a wave, in every lane.
__device__ __forceinline__ float wave_max(float x) {
    x = fmax_nn(x, dpp<0xB1>(x));
    x = fmax_nn(x, dpp<0x4E>(x));
    x = fmax_nn(x, dpp<0x141>(x));
    x = fmax_nn(x, dpp<0x140>(x));
    return xrow_max(x);
}

__device__ __forceinline__ float half_lo(const uint32_t x) { return f16_to_f32(static_cast<uint16_t>(x & 0xffffu)); }
__device__ __forceinline__ float half_hi(const uint32_t x) { return f16_to_f32(static_cast<uint16_t>(x >> 16)); }

// The prefix's tiers for one KV head.
struct Tiers {
    const float* dk;
    const float* dv;
    const uint32_t* kp;
    const char* ks;
    const char* kz;
    const uint32_t* vp;
    const char* vs;
    const char* vz;
    const int64_t* ids;
    int nd, slots;    // FP32 tokens, packed slots
};

__device__ __forceinline__ Tiers tiers_of(const SharedArgs& a, const int kvh) {
    const tt_decode_seq& d = a.prefix;
    const size_t m = a.meta_fp16 ? 2 : 4;
    Tiers t;
    t.dk = d.dense_K + static_cast<size_t>(kvh) * a.D;
    t.dv = d.dense_V + static_cast<size_t>(kvh) * a.D;
    t.kp = reinterpret_cast<const uint32_t*>(d.PBS_K_Packed) + static_cast<size_t>(kvh) * a.D;
    t.ks = static_cast<const char*>(d.PBS_K_Scales) + kvh * a.D * m;
    t.kz = static_cast<const char*>(d.PBS_K_Zeroes) + kvh * a.D * m;
    t.vp = reinterpret_cast<const uint32_t*>(d.PBS_V_Packed) + static_cast<size_t>(kvh) * (a.D / 16);
    t.vs = static_cast<const char*>(d.PBS_V_Scales) + kvh * m;
    t.vz = static_cast<const char*>(d.PBS_V_Zeroes) + kvh * m;
    t.ids = d.PBS_token_ids;
    t.nd = d.dense_count;
    t.slots = d.num_blocks * a.kgs;
    return t;
}

// Orders LDS accesses over the workgroup without waiting for loads from memory.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The largest k and v (>= 0) of a workgroup of WM waves, in every lane, through `lds`, which is free behind the next barrier.
template <int WM>
__device__ __forceinline__ float2 group_max(float k, float v, char* lds, const int wave, const int lane) {
    float2* x = reinterpret_cast<float2*>(lds);
    k = wave_max(k);
    v = wave_max(v);
    if (lane == 0) x[wave] = make_float2(k, v);
    lds_barrier();
    float2 m = x[0];
#pragma unroll
    for (int i = 1; i < WM; ++i) {
        const float2 y = x[i];
        m = make_float2(fmax_nn(m.x, y.x), fmax_nn(m.y, y.y));
    }
    return m;
}

typedef uint32_t un_u4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t un_u2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename MetaT>
using MetaBits = std::conditional_t<sizeof(MetaT) == 2, uint16_t, uint32_t>;

// Asks for an order of the block's instructions: a few vector ones behind each
// of M matrix ones, whose pipe then runs while they issue. (Left alone the
// compiler puts all matrix instructions first.)
template <int M>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < M; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // VALU
    }
}

typedef float mf_f16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ mf_f16 mfma32x32x16(const mf_u4 a, const mf_u4 b, const mf_f16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(mf_h8, a), __builtin_bit_cast(mf_h8, b), c, 0, 0, 0);
}

// For operands that are never NaN (fmaxf would quiet those it cannot see the origin of).
__device__ __forceinline__ float max3(const float a, const float b, const float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Loads from a uniform base at a 32-bit lane offset in bytes.
template <typename T>
__device__ __forceinline__ T load_at(const void* base, const uint32_t off) {
    return *reinterpret_cast<const T*>(static_cast<const char*>(base) + off);
}

// A loaded value that is used from here on: its uses (and the wait for it) do not move further up.
template <typename T>
__device__ __forceinline__ void pin(T& x) {
    asm volatile("" : "+v"(x));
}
__device__ __forceinline__ void pin(mf_u4& x, const int e) {
    uint32_t y = x[e];
    asm volatile("" : "+v"(y));
    x[e] = y;
}

// Ends a group of instructions that the scheduler may not mix with the next.
__device__ __forceinline__ void slot_end() { __builtin_amdgcn_sched_barrier(0); }

// Row n of a wave's 32, the lane's half h of each 16 channels.
struct Row {
    bool live;
    int seq, head;
};
__device__ __forceinline__ Row row_of(const SharedArgs& a, const int kvh, const int rn, const int rows) {
    const int G = a.Hq / a.Hkv;
    const bool live = rn < rows;
    return Row{live, live ? rn / G : 0, kvh * G + (live ? rn % G : 0)};
}

// Q' = Q 2^(12 - e), e the exponent of the row's largest value, in parts: channels 16 s + 8 h .. + 7. Returns the log2 units per
// unit of the product.
template <int ST>
__device__ __forceinline__ float queries(const SharedArgs& a, const Row& row, const int h, const float neg1, mf_u4 (&qh)[ST],
                                         mf_u4 (&ql)[ST]) {
    const int D = a.D;
    const float* q = global_ptr(a.seqs[row.seq].Q) + static_cast<size_t>(row.head) * D;
    float mx = 0.0f;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        const int c = min(16 * s + 8 * h, D - 8);
        qh[s] = *reinterpret_cast<const un_u4*>(q + c);
        ql[s] = *reinterpret_cast<const un_u4*>(q + c + 4);
    }
#pragma unroll
    for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!row.live || 16 * s + 8 * h >= D) qh[s][j] = ql[s][j] = 0u;
            mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(qh[s][j])), fabsf(__uint_as_float(ql[s][j]))));
        }
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const int e = (mx > 0.0f) ? __builtin_amdgcn_frexp_expf(mx) : 0;
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        uint2 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const mf_u4 x = j < 2 ? qh[s] : ql[s];
            p[j] = tt::parts(__builtin_amdgcn_ldexpf(__uint_as_float(x[2 * (j & 1)]), 12 - e),
                         __builtin_amdgcn_ldexpf(__uint_as_float(x[2 * (j & 1) + 1]), 12 - e), neg1);
        }
        qh[s] = mf_u4{p[0].x, p[1].x, p[2].x, p[3].x};
        ql[s] = mf_u4{p[0].y, p[1].y, p[2].y, p[3].y};
    }
    return __builtin_amdgcn_ldexpf(a.scale2, e - 16);
}

// The softmax of a tile's logits d (lane (h, n): tokens 8 (r / 4) + 4 h + r % 4 of row n; `mask` its attended tokens, c log2 units per
// unit, `meta` packed V's scales and zeros) into P, times V's scale where that is packed, in parts as the PV A operand.
struct Soft {
    float mr = -3.0e38f, l = 0.0f, pz = 0.0f;  // reference, sum, sum of P times the centred zero
};
template <int DC, bool PACKED, typename F>
__device__ __forceinline__ void softmax32(Soft& s_, mf_f16& d, mf_f16 (&acc)[DC], const uint32_t mask, const float c, const char* meta,
                                          const int lane, const float neg1, mf_u4 (&ph)[2], mf_u4 (&pl)[2], F&& before) {
    float &mr = s_.mr, &l = s_.l, &pz = s_.pz;
    const int h = lane >> 5;
    auto now = [](int x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    if (mask != 0xffffffffu) {
        const uint32_t mine = mask >> (4 * (now(lane) >> 5));
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] = ((mine >> (8 * (r >> 2) + (r & 3))) & 1u) ? d[r] : kNegInf;
    }
    float mx = max3(max3(d[0], d[1], d[2]), max3(d[3], d[4], d[5]), max3(d[6], d[7], d[8]));
    mx = max3(mx, max3(d[9], d[10], d[11]), max3(d[12], d[13], max3(d[14], d[15], d[15])));
    mx = __builtin_fmaf(mx, c, -kUp);
    // the reference moves only when a row's maximum passes it by more than the slack
    if (__ballot(mx > mr + kSlack)) {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        const bool up = mx > mr + kSlack;
        const float mn = up ? mx : mr;
        const float al = up ? __builtin_amdgcn_exp2f(mr - mn) : 1.0f;
        l *= al;
        pz *= al;
        const int from = 16 * (now(lane) >> 5);  // bytes: the lane group's first row
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float ar = __int_as_float(__builtin_amdgcn_ds_bpermute(from + 4 * (8 * (r >> 2) + (r & 3)), __float_as_int(al)));
#pragma unroll
            for (int s = 0; s < DC; ++s) acc[s][r] *= ar;
        }
        mr = mn;
    }
    before();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mf_f4 vs, vz;
        if constexpr (PACKED) {
            vs = *reinterpret_cast<const mf_f4*>(meta + 32 * j + 16 * h);
            vz = *reinterpret_cast<const mf_f4*>(meta + 128 + 32 * j + 16 * h);
        }
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(d[4 * j + r], c, -mr));
        l += (p[0] + p[1]) + (p[2] + p[3]);
        if constexpr (PACKED) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pz = __builtin_fmaf(p[r], vz[r], pz);
                p[r] *= vs[r];
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint2 y = tt::parts(p[2 * x], p[2 * x + 1], neg1);
            ph[j >> 1][2 * (j & 1) + x] = y.x;
            pl[j >> 1][2 * (j & 1) + x] = y.y;
        }
    }
}

// Writes a wave's partial, of rows row0 .. + 31. (NC: packed V's codes are 4^(c % NC) times too large.)
template <int DC, int NC, bool PACKED>
__device__ __forceinline__ void store32(const SharedArgs& a, const Row& row, const Soft& s_, const mf_f16 (&acc)[DC], const int v_exp,
                                        const int lane, const int row0, const int rows, const int slot) {
    const int D = a.D, n = lane & 31, h = lane >> 5;
    // The partial in units of V: acc holds 16 V 2^-v_exp (FP32 tiles), or 2 4^(c % NC) of it without the centred zero.
    auto both = [&](const float x) {  // a row's sum over its two lanes
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    };
    const float l = both(s_.l);
    const float z = PACKED ? __builtin_amdgcn_ldexpf(both(s_.pz), v_exp) : 0.0f;
    const float back = __builtin_amdgcn_ldexpf(1.0f, v_exp - (PACKED ? 1 + 2 * (n & (NC - 1)) : 4));
    // row n's partial, behind its sequence's own slots
    const int ns = a.slot_base[row.seq + 1] - a.slot_base[row.seq];
    const uint32_t pi = static_cast<uint32_t>(a.slot_base[row.seq] * a.Hq + row.head * ns + (ns - a.prefix_slots + slot));
    if (h == 0 && row.live) {
        a.ml[2 * static_cast<size_t>(pi)] = l > 0.0f ? s_.mr : kNegInf;
        a.ml[2 * static_cast<size_t>(pi) + 1] = l;
    }
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int first = 4 * (ln >> 5);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int r_ = 8 * (r >> 2) + first + (r & 3);
        const float zr = PACKED ? __shfl(z, r_, 64) : 0.0f;
        const uint32_t pr = static_cast<uint32_t>(__shfl(static_cast<int>(pi), r_, 64));
        if (row0 + r_ >= rows) continue;
        float* o = a.acc + static_cast<size_t>(pr) * D + n;
#pragma unroll
        for (int s = 0; s < DC; ++s)
            if (32 * s + n < D) o[32 * s] = __builtin_fmaf(acc[s][r], back, zr);
    }
}

// One workgroup's share [t0, t1) of the prefix's tiles of one kind, for rows row0 .. of one KV head, head_dim up to
// 32 DC. WM waves of 32 rows each, on the same tile.
//
//   QK  A = K (32 tokens x 16 channels), B = Q (16 channels x 32 rows): lane (h = lane / 32, n = lane % 32) receives
//       tokens 8 (r / 4) + 4 h + r % 4 of row n, r < 16.
//   PV  A = P (32 rows x 16 tokens), B = V (16 tokens x 32 channels): a lane's values r = 8 j .. 8 j + 7 are its A operand
//       of step j, so V's tokens lie in LDS in the order position 16 j + 8 h + i <-> token 16 j + 8 (i / 4) + 4 h + i % 4.
//
// While the matrix cores multiply Q with K of tile k, the VALU stages tile
// k + 1, whose loads went out a tile earlier. One barrier per tile. The order of
// the two kinds of instructions is written out (a matrix instruction, then
// vector ones while it runs): left alone the compiler puts all matrix
// instructions first, each behind the wait for its LDS operands.
template <int DC, int WM, bool PACKED, typename MetaT>
__device__ __forceinline__ void shared_body(const SharedArgs& a, char* lds, const Tiers& t, const int kvh,
                                            const int row0, const int rows, const int t0, const int t1,
                                            const int slot) {
    using L = TileLds<DC>;
    constexpr bool F16M = sizeof(MetaT) == 2;
    constexpr int ST = 2 * DC;  // QK steps
    float neg1 = -1.0f;
    asm("" : "+s"(neg1));
    auto parts = [&](const float x0, const float x1) { return tt::parts(x0, x1, neg1); };
    const int lane = threadIdx.x & 63;
    const int wave = scalar(static_cast<int>(threadIdx.x) >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int D = a.D;
    const uint32_t stride = static_cast<uint32_t>(a.Hkv) * D;  // elements between tokens (blocks) of a head
    // A unit is 64 lanes x (4 tokens x 4 channels) of a tile: 32 channels. Every wave stages the same share of a K and of
    // a V unit: NT tokens and NC channels of each lane's. (With three units some waves repeat the last one's.)
    constexpr int UNITS = DC == 3 ? 4 : DC, SHARES = WM / UNITS, NT = 4 / SHARES, NC = 4 / SHARES;
    const int unit = min(wave % UNITS, DC - 1), part = wave / UNITS;
    // K: lane = (token quad, channel quad); V the other way round, so that the
    // writes of V's transposed rows spread over the banks.
    const int ktq = lane >> 3, kcq = lane & 7;
    const int vtq = lane & 7, vcq = lane >> 3;
    const int kc = 32 * unit + 4 * kcq, vc = 32 * unit + 4 * vcq;  // first channels
    const int kt0 = 4 * ktq + NT * part;                           // first token

    // The tile in flight, as it lies in memory.
    mf_u4 kx[PACKED ? 3 : NT];        // packed: words, scale, zero; FP32: tokens
    uint32_t vx[4][PACKED ? 1 : NC];  // packed: words of 4 tokens; FP32: 4 tokens' channels
    uint2 idv = make_uint2(0u, 0u);
    uint32_t vm = 0u;                 // packed: V scale (lanes 0-31) or zero (lanes 32-63) of token lane % 32
    // A value as one of its own: what is computed from it inside the loop is not kept in registers over it.
    auto now = [&](auto x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    // A tile of 32 tokens that passes the end of the tier is read from 32 before it, its tokens of the tile before masked:
    // so the lanes' offsets from a tile's start are the same for all tiles. (Of a tier shorter than a tile, the tokens
    // past the last repeat it.)
    const int total = PACKED ? t.slots : t.nd;
    auto start_of = [&](const int tile) { return max(min(kTile * tile, total - kTile), 0); };
    uint32_t o_id = 0u, o_km = 0u, o_vm = 0u, o_k, o_v;  // (those of K and V: the lane's first token)
    uint32_t k_end = 0u, v_end = 0u;                     // FP32: the last token's
    {
        const int last = min(total, kTile) - 1;
        const uint32_t ck = min(kc, D - 4), cv = min(vc, D - 4);
        if constexpr (PACKED) {
            constexpr uint32_t M = sizeof(MetaT);
            o_id = 8u * min(n, last);
            o_k = 4u * ((min(4 * ktq, last) >> 4) * stride + ck);
            o_km = M * (a.kgs == 32 ? ck : o_k / 4u);
            o_vm = static_cast<uint32_t>(min(n, last)) * a.Hkv * M;
            o_v = 4u * (min(4 * vtq, last & ~3) * (stride / 16) + (cv >> 4));
        } else {
            o_k = 4u * (kt0 * stride + ck);
            k_end = 4u * (last * stride + ck);
            o_v = 4u * (4 * vtq * stride + cv + NC * part);
            v_end = 4u * (last * stride + cv + NC * part);
        }
    }
    auto fetch = [&](const int tile) {
        const int s0 = start_of(tile);
        if constexpr (PACKED) {
            constexpr uint32_t M = sizeof(MetaT);
            const size_t kb = static_cast<size_t>(a.kgs == 32 ? s0 >> 5 : s0 >> 4) * stride * M;
            idv = load_at<uint2>(t.ids + s0, o_id);
            kx[0] = load_at<un_u4>(t.kp + static_cast<size_t>(s0 >> 4) * stride, o_k);
            if constexpr (!F16M) {
                kx[1] = load_at<un_u4>(t.ks + kb, o_km);
                kx[2] = load_at<un_u4>(t.kz + kb, o_km);
            } else {
                const un_u2 ps = load_at<un_u2>(t.ks + kb, o_km), pz = load_at<un_u2>(t.kz + kb, o_km);
                kx[1] = mf_u4{ps[0], ps[1], pz[0], pz[1]};
            }
            // V's scales in lanes 0-31, its zeros in lanes 32-63
            const char* from = (lane < 32 ? t.vs : t.vz) + static_cast<size_t>(s0) * a.Hkv * M;
            vm = load_at<MetaBits<MetaT>>(from, o_vm);
            const size_t words = stride / 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) vx[j][0] = load_at<uint32_t>(t.vp + (s0 + j) * words, o_v);
        } else {
            const float* keys = t.dk + static_cast<size_t>(s0) * stride;
            const float* values = t.dv + static_cast<size_t>(s0) * stride;
            const uint32_t ok = now(o_k), ov = now(o_v);
#pragma unroll
            for (int j = 0; j < NT; ++j) kx[j] = load_at<un_u4>(keys, min(ok + 4u * j * stride, k_end));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t off = min(ov + 4u * j * stride, v_end);
                if constexpr (NC == 1) {
                    vx[j][0] = load_at<uint32_t>(values, off);
                } else {
                    typedef uint32_t un_nc __attribute__((ext_vector_type(NC), aligned(4)));
                    const un_nc y = load_at<un_nc>(values, off);
#pragma unroll
                    for (int e = 0; e < NC; ++e) vx[j][e] = y[e];
                }
            }
        }
    };
    // Bit j: token j of the tile is attended (packed: of the K tile in flight).
    auto mask_of = [&](const int tile) -> uint32_t {
        const uint32_t in = total < kTile ? (1u << total) - 1u : 0xffffffffu << (kTile * tile - start_of(tile));
        if constexpr (PACKED) return static_cast<uint32_t>(__ballot((idv.x & idv.y) != 0xffffffffu)) & in;
        return in;
    };

    float* peak = reinterpret_cast<float*>(lds + 2 * L::BYTES);  // [tile's parity][key, value]
    // A tile's largest key or value where it asks for another scale: too large for f16 at this one, or (first) any.
    // The peaks only grow and so do the exponents after the first: none is ever cleared. They are looked at once the
    // tile's logits are there, which then are not used if they ask for another scale.
    // Positive floats order like their bits. (An infinity has no scale that helps: it is left to make NaN of what
    // reads it.)
    auto report = [&](const float x, const float back, const bool first, float* to) {
        if ((x >= kLimit || (first && x > 0.0f)) && x < __builtin_huge_valf())
            atomicMax(reinterpret_cast<int*>(to), __float_as_int(fminf(x * back, 3.0e38f)));
    };

    // Staging, in pieces to go between matrix instructions: f16 parts of the fetched K times 2^(4 - k_exp) ...
    float ksc[4], kzr[4], kmx, vmx;
    uint32_t kcodes, vcodes[2];
    auto k_scale = [&](const int e, const uint32_t mask, const float by) {
        // no attended token: the block's scale and zero may be anything
        const bool any = ((mask >> (4 * ktq)) & 15u) != 0u && kc < D;
        if constexpr (PACKED) {
            pin(kx[1], F16M ? e >> 1 : e);
            pin(kx[F16M ? 1 : 2], F16M ? 2 + (e >> 1) : e);
            if constexpr (F16M) {
                const uint32_t hs = kx[1][e >> 1], hz = kx[1][2 + (e >> 1)];
                ksc[e] = (e & 1) ? half_hi(hs) : half_lo(hs);
                kzr[e] = (e & 1) ? half_hi(hz) : half_lo(hz);
            } else {
                ksc[e] = __uint_as_float(kx[1][e]);
                kzr[e] = __uint_as_float(kx[2][e]);
            }
            ksc[e] = any ? ksc[e] * by : 0.0f;
            kzr[e] = any ? kzr[e] * by : 0.0f;
            kmx = fmaxf(kmx, fmaxf(fabsf(kzr[e]), fabsf(__builtin_fmaf(3.0f, ksc[e], kzr[e]))));
        }
    };
    auto k_gather = [&]() {
#pragma unroll
        for (int e = 0; e < 4; ++e) pin(kx[0], e);
        // the quad's codes, one byte per channel, from the lane's first token on
        const uint32_t b = 0x0c0c0400u + 0x0101u * (ktq & 3);
        const uint32_t lo = __builtin_amdgcn_perm(kx[0][1], kx[0][0], b);
        const uint32_t hi = __builtin_amdgcn_perm(kx[0][3], kx[0][2], b);
        kcodes = (lo | (hi << 16)) >> (2 * NT * part);
    };
    auto k_token = [&](char* tl, const int j, const uint32_t mask, const float by) {
        float x[4];
        if constexpr (PACKED) {
            uint32_t y = (kcodes >> (2 * j)) & 0x03030303u;
            asm("" : "+v"(y));  // (or every code is extracted by an instruction of its own)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(static_cast<float>((y >> (8 * e)) & 0xffu), ksc[e], kzr[e]);
        } else {
            const bool in = ((mask >> (kt0 + j)) & 1u) && kc < D;
#pragma unroll
            for (int e = 0; e < 4; ++e) pin(kx[j], e);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = in ? __uint_as_float(kx[j][e]) * by : 0.0f;
                kmx = fmaxf(kmx, fabsf(x[e]));
            }
        }
        const uint2 p = parts(x[0], x[1]), q = parts(x[2], x[3]);
        char* d = tl + (kt0 + j) * L::KS + 2 * kc;
        *reinterpret_cast<uint2*>(d + L::KHI) = make_uint2(p.x, q.x);
        *reinterpret_cast<uint2*>(d + L::KLO) = make_uint2(p.y, q.y);
    };
    // ... and V: packed, the centred codes (2 q - 3) 4^(c % NC), exact, of channels c; FP32, f16 parts of V 2^(4 - v_exp).
    // Token quad vtq in its place in the PV order.
    const int vplace = 32 * (vtq >> 2) + 16 * (vtq & 1) + 8 * ((vtq >> 1) & 1);  // bytes
    auto v_gather = [&]() {
#pragma unroll
        for (int j = 0; j < 4; ++j) pin(vx[j][0]);
        // the codes of the lane's first channel at bit 1 of each half
        const uint32_t b = 0x0c040c00u + 0x00010001u * (vcq & 3);
        vcodes[0] = (__builtin_amdgcn_perm(vx[1][0], vx[0][0], b) << 1) >> (2 * NC * part);
        vcodes[1] = (__builtin_amdgcn_perm(vx[3][0], vx[2][0], b) << 1) >> (2 * NC * part);
    };
    auto v_channel = [&](char* tl, const int k, const uint32_t mask, const float by) {
        char* d = tl + (vc + NC * part + k) * L::VS + vplace;
        if constexpr (PACKED) {
            // channels past head_dim hold codes of others, in columns that are not stored
            const _Float16 c = static_cast<_Float16>(1024.0f + 3.0f * static_cast<float>(1 << (2 * k)));
            const mf_h2 off = {c, c};
            const uint32_t mk = 0x00060006u << (2 * k);
            const mf_h2 z0 = __builtin_bit_cast(mf_h2, (vcodes[0] & mk) | 0x64006400u) - off;
            const mf_h2 z1 = __builtin_bit_cast(mf_h2, (vcodes[1] & mk) | 0x64006400u) - off;
            *reinterpret_cast<uint2*>(d + L::V) =
                make_uint2(__builtin_bit_cast(uint32_t, z0), __builtin_bit_cast(uint32_t, z1));
        } else {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                pin(vx[j][k]);
                y[j] = ((mask >> (4 * vtq + j)) & 1u) && vc < D ? __uint_as_float(vx[j][k]) * by : 0.0f;
                vmx = fmaxf(vmx, fabsf(y[j]));
            }
            const uint2 p = parts(y[0], y[1]), q = parts(y[2], y[3]);
            *reinterpret_cast<uint2*>(d + L::V) = make_uint2(p.x, q.x);
            *reinterpret_cast<uint2*>(d + L::VLO) = make_uint2(p.y, q.y);
        }
    };
    // Packed: V's scale 2^-v_exp and the zero of the centred codes, vz + 1.5 vs, of the tile's tokens, zeros where masked.
    // (Every wave writes the same.)
    auto stage_meta = [&](char* tl, const uint32_t mask, const int ve) {
        pin(vm);
        const float x = F16M ? half_lo(vm) : __uint_as_float(vm);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        float y = lane < 32 ? x : __builtin_fmaf(1.5f, __uint_as_float(sw[0]), x);
        y = ((mask >> n) & 1u) ? __builtin_amdgcn_ldexpf(y, -ve) : 0.0f;
        reinterpret_cast<float*>(tl + L::VMETA)[lane] = y;
        // a scale up to 2 2^v_exp stays in reach (P <= 2^14): in units of kLimit / 2
        vmx = lane < 32 ? fabsf(y) * (0.5f * kLimit) : 0.0f;
    };

    fetch(t0);  // its loads go out before the queries'
    float2 top;  // the first tile's largest key and value
    {
        const uint32_t m = mask_of(t0);
        kmx = vmx = 0.0f;
        if constexpr (PACKED) {
#pragma unroll
            for (int e = 0; e < 4; ++e) k_scale(e, m, 1.0f);
            vmx = lane < 32 && ((m >> n) & 1u) ? fabsf(F16M ? half_lo(vm) : __uint_as_float(vm)) : 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    kmx = fmaxf(kmx, ((m >> (kt0 + j)) & 1u) && kc < D ? fabsf(__uint_as_float(kx[j][e])) : 0.0f);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < NC; ++e)
                    vmx = fmaxf(vmx, ((m >> (4 * vtq + j)) & 1u) && vc < D ? fabsf(__uint_as_float(vx[j][e])) : 0.0f);
        }
        top = group_max<WM>(kmx, vmx, lds, wave, lane);
    }
    const Row row = row_of(a, kvh, row0 + 32 * wave + n, rows);
    const bool rowed = row0 + 32 * wave < rows;  // a wave without rows only stages (and multiplies zeros with K)
    mf_u4 qh[ST], ql[ST];
    const float crow = queries<ST>(a, row, h, neg1, qh, ql);

    mf_f16 acc[DC];
    Soft st;
#pragma unroll
    for (int s = 0; s < DC; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[s][r] = 0.0f;
    // Exponents of the scales of K and V (uniform over the workgroup), and whether no tile has set them yet.
    int k_exp = exponent(top.x, 8), v_exp = exponent(top.y, PACKED ? 0 : 8);
    bool kfirst = !__ballot(top.x > 0.0f), vfirst = !__ballot(top.y > 0.0f);
    if (threadIdx.x < 4) peak[threadIdx.x] = 0.0f;

    // At the top of the loop tile k is staged and tile k + 1 in flight. `again`: tile k is in flight and has to be staged,
    // at the start or with other exponents; its products are not used then.
    int again = 1;
    asm("" : "+s"(again));  // (or the compiler makes a loop of its own of the start)
    uint32_t mask = 0u;  // of tile k
    int k = t0;
#pragma unroll 1
    do {
        lds_barrier();
        const float pk_k = peak[2 * (k & 1)], pk_v = peak[2 * (k & 1) + 1];
        const int next = min(again ? k : k + 1, t1 - 1);  // the tile in flight
        const char* tl = lds + (k & 1) * L::BYTES;
        uint32_t mnext = 0u;
        mf_f16 d;
        {
            // QK of tile k, between its instructions the tile in flight to LDS.
            const char* kl = tl + n * L::KS + 16 * h;
            const int to = again ? k & 1 : (k + 1) & 1;
            char* dst = lds + to * L::BYTES;
            const float kby = __builtin_amdgcn_ldexpf(16.0f, -k_exp), vby = __builtin_amdgcn_ldexpf(16.0f, -v_exp);
            constexpr int PIECES = PACKED ? 8 + NT + NC : 1 + NT + NC, SLOTS = 3 * ST;
            auto piece = [&](const int i) {
                if (i == 0) {
                    pin(idv.x);
                    pin(idv.y);
                    mnext = mask_of(next);
                    kmx = vmx = 0.0f;
                } else if (PACKED && i < 5) {
                    k_scale(i - 1, mnext, kby);
                } else if (PACKED && i == 5) {
                    k_gather();
                } else if (i < (PACKED ? 6 : 1) + NT) {
                    k_token(dst, i - (PACKED ? 6 : 1), mnext, kby);
                } else if (PACKED && i == 6 + NT) {
                    v_gather();
                } else if (PACKED && i == 7 + NT) {
                    stage_meta(dst, mnext, v_exp);
                } else {
                    v_channel(dst, i - (PACKED ? 8 : 1) - NT, mnext, vby);
                }
            };
            mf_u4 kh[2], kw[2];
            auto load_k = [&](const int s) {
                kh[s & 1] = *reinterpret_cast<const mf_u4*>(kl + L::KHI + 32 * s);
                kw[s & 1] = *reinterpret_cast<const mf_u4*>(kl + L::KLO + 32 * s);
            };
            load_k(0);
            slot_end();
#pragma unroll
            for (int r = 0; r < 16; ++r) d[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                const int s = i / 3;
                if (i % 3 == 0 && s + 1 < ST) load_k(s + 1);
                d = mfma32x32x16(i % 3 == 2 ? kw[s & 1] : kh[s & 1], i % 3 == 0 ? ql[s] : qh[s], d);
#pragma unroll
                for (int o = i * PIECES / SLOTS; o < (i + 1) * PIECES / SLOTS; ++o) piece(o);
                slot_end();
            }
            if (__ballot(fmaxf(kmx, vmx) >= kLimit) || kfirst || vfirst) {
                report(kmx, __builtin_amdgcn_ldexpf(0.0625f, k_exp), kfirst, peak + 2 * to);
                report(vmx, __builtin_amdgcn_ldexpf(PACKED ? 2.0f / kLimit : 0.0625f, v_exp), vfirst, peak + 2 * to + 1);
            }
        }
        int ahead = again ? k + 1 : k + 2;  // the tile to fetch
        const int skip = again;
        if (!again && __ballot(fmaxf(pk_k, pk_v) > 0.0f)) {
            int kn = k_exp, vn = v_exp;
            if (__ballot(pk_k > 0.0f)) {
                const int e = exponent(pk_k, 8);  // (a peak past the limit asks for 4 more at least)
                if (e - 3 > k_exp || kfirst) kn = e;
                kfirst = false;
            }
            if (__ballot(pk_v > 0.0f)) {
                const int e = exponent(pk_v, PACKED ? 0 : 8);
                if (e - (PACKED ? 1 : 3) > v_exp || vfirst) vn = e;
                vfirst = false;
            }
            if (kn != k_exp || vn != v_exp) {
                const float f = __builtin_amdgcn_ldexpf(1.0f, v_exp - vn);
                st.pz *= f;
#pragma unroll
                for (int s = 0; s < DC; ++s) acc[s] *= f;
                k_exp = kn;
                v_exp = vn;
                again = 2;
                ahead = k;
            }
        }
        // (The one place in the loop that fetches: of several, copies would be made, which wait for the loads.)
        fetch(min(ahead, t1 - 1));
        again = again == 2 ? 1 : 0;
        if (rowed && !(skip | again)) {
            mf_u4 vh[2], vw[2];
            auto load_v = [&](const int s) {  // step s: channels 32 (s / 2) .., tokens of half s % 2
                const char* x = tl + (32 * (s >> 1) + n) * L::VS + 32 * (s & 1) + 16 * h;
                vh[s & 1] = *reinterpret_cast<const mf_u4*>(x + L::V);
                if constexpr (!PACKED) vw[s & 1] = *reinterpret_cast<const mf_u4*>(x + L::VLO);
            };
            mf_u4 ph[2], pl[2];
            softmax32<DC, PACKED>(st, d, acc, mask, __builtin_amdgcn_ldexpf(crow, k_exp), tl + L::VMETA, lane, neg1, ph, pl,
                                  [&]() { load_v(0); });
            constexpr int PR = PACKED ? 2 : 3, SLOTS = 2 * DC * PR;
            slot_end();
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                const int s = i / PR, q = i % PR;
                if (q == 0 && s + 1 < 2 * DC) load_v(s + 1);
                acc[s >> 1] = mfma32x32x16(q == 0 ? pl[s & 1] : ph[s & 1], !PACKED && q == 1 ? vw[s & 1] : vh[s & 1], acc[s >> 1]);
                slot_end();
            }
        }
        mask = mnext;
        k += skip | again ? 0 : 1;
    } while (k < t1);

    store32<DC, NC, PACKED>(a, row, st, acc, v_exp, lane, row0 + 32 * wave, rows, slot);
}

// One wave's share of the tiles for at most 32 rows of one KV head, where there are no rows for more waves: each stages
// whole tiles of its own, without a barrier, in its own part of the LDS. K of a tile is staged between the PV instructions
// of the one before, V between its own QK ones, so that one buffer does. Scales change before a tile is staged. One wave per
// SIMD, with up to 400 registers: the VALU, which unpacks a tile for 32 rows only, takes more of it than the matrix cores (8
// sequences behind 16k tokens, 32/32 heads of 80: 16 to 17 tiles per wave, 56 us in all).
template <int DC, bool PACKED, typename MetaT>
__device__ __forceinline__ void lone_body(const SharedArgs& a, char* lds, const Tiers& t, const int kvh, const int row0,
                                          const int rows, const int t0, const int t1, const int slot) {
    using L = TileLds<DC>;
    constexpr bool F16M = sizeof(MetaT) == 2;
    constexpr int ST = 2 * DC;
    float neg1 = -1.0f;
    asm("" : "+s"(neg1));
    auto parts = [&](const float x0, const float x1) { return tt::parts(x0, x1, neg1); };
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int D = a.D;
    const uint32_t stride = static_cast<uint32_t>(a.Hkv) * D;
    const int ktq = lane >> 3, kcq = lane & 7, vtq = lane & 7, vcq = lane >> 3;  // as for the larger groups, unit u: channels 32 u ..
    const int total = PACKED ? t.slots : t.nd;
    auto start_of = [&](const int tile) { return max(min(kTile * tile, total - kTile), 0); };
    const int last = min(total, kTile) - 1;

    uint32_t kx[DC][PACKED ? 12 : 16], vx[DC][PACKED ? 4 : 16], vm = 0u;
    uint2 idv = make_uint2(0u, 0u);
    auto get4 = [&](uint32_t* to, const void* base, const uint32_t off) {
        const un_u4 y = load_at<un_u4>(base, off);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = y[e];
    };
    auto fetch_k = [&](const int tile) {
        const int s0 = start_of(tile);
        constexpr uint32_t M = sizeof(MetaT);
        if constexpr (PACKED) idv = load_at<uint2>(t.ids + s0, 8u * min(n, last));
#pragma unroll
        for (int u = 0; u < DC; ++u) {
            const uint32_t ck = min(32 * u + 4 * kcq, D - 4);
            if constexpr (PACKED) {
                const uint32_t kw = (min(4 * ktq, last) >> 4) * stride + ck, km = M * (a.kgs == 32 ? ck : kw);
                const size_t kb = static_cast<size_t>(a.kgs == 32 ? s0 >> 5 : s0 >> 4) * stride * M;
                get4(kx[u], t.kp + static_cast<size_t>(s0 >> 4) * stride, 4u * kw);
                if constexpr (!F16M) {
                    get4(kx[u] + 4, t.ks + kb, km);
                    get4(kx[u] + 8, t.kz + kb, km);
                } else {
                    const un_u2 ps = load_at<un_u2>(t.ks + kb, km), pz = load_at<un_u2>(t.kz + kb, km);
                    kx[u][4] = ps[0];
                    kx[u][5] = ps[1];
                    kx[u][6] = pz[0];
                    kx[u][7] = pz[1];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    get4(kx[u] + 4 * j, t.dk + static_cast<size_t>(s0) * stride, 4u * (min(4 * ktq + j, last) * stride + ck));
            }
        }
    };
    auto fetch_v = [&](const int tile) {
        const int s0 = start_of(tile);
        constexpr uint32_t M = sizeof(MetaT);
        if constexpr (PACKED) {
            const char* from = (lane < 32 ? t.vs : t.vz) + static_cast<size_t>(s0) * a.Hkv * M;
            vm = load_at<MetaBits<MetaT>>(from, static_cast<uint32_t>(min(n, last)) * a.Hkv * M);
        }
#pragma unroll
        for (int u = 0; u < DC; ++u) {
            const uint32_t cv = min(32 * u + 4 * vcq, D - 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (PACKED)
                    vx[u][j] = load_at<uint32_t>(t.vp + static_cast<size_t>(s0) * (stride / 16),
                                                 4u * (min(4 * vtq + j, last) * (stride / 16) + (cv >> 4)));
                else
                    get4(vx[u] + 4 * j, t.dv + static_cast<size_t>(s0) * stride, 4u * (min(4 * vtq + j, last) * stride + cv));
            }
        }
    };
    auto mask_of = [&](const int tile) -> uint32_t {
        const uint32_t in = total < kTile ? (1u << total) - 1u : 0xffffffffu << (kTile * tile - start_of(tile));
        if constexpr (PACKED) return static_cast<uint32_t>(__ballot((idv.x & idv.y) != 0xffffffffu)) & in;
        return in;
    };

    int k_exp = 0, v_exp = 0;
    bool kfirst = true, vfirst = true;
    Soft st;
    mf_f16 acc[DC];
#pragma unroll
    for (int s = 0; s < DC; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[s][r] = 0.0f;

    // K's scales and zeros of the fetched tile (packed), and its exponent: what passes the limit, or comes first, sets it.
    float ksc[PACKED ? DC : 1][4], kzr[PACKED ? DC : 1][4];
    auto ready_k = [&](const uint32_t mask) {
        float mx = 0.0f;
#pragma unroll
        for (int u = 0; u < DC; ++u) {
            const int kc = 32 * u + 4 * kcq;
            if constexpr (PACKED) {
                const bool any = ((mask >> (4 * ktq)) & 15u) != 0u && kc < D;  // else they may be anything
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t hs = kx[u][4 + (F16M ? e >> 1 : e)], hz = kx[u][F16M ? 6 + (e >> 1) : 8 + e];
                    const float sc = F16M ? ((e & 1) ? half_hi(hs) : half_lo(hs)) : __uint_as_float(hs);
                    const float zr = F16M ? ((e & 1) ? half_hi(hz) : half_lo(hz)) : __uint_as_float(hz);
                    ksc[u][e] = any ? sc : 0.0f;
                    kzr[u][e] = any ? zr : 0.0f;
                    mx = fmaxf(mx, fmaxf(fabsf(kzr[u][e]), fabsf(__builtin_fmaf(3.0f, ksc[u][e], kzr[u][e]))));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    mx = fmaxf(mx, ((mask >> (4 * ktq + i / 4)) & 1u) && kc < D ? fabsf(__uint_as_float(kx[u][i])) : 0.0f);
            }
        }
        if (__ballot(__builtin_amdgcn_ldexpf(mx, 4 - k_exp) >= kLimit || (kfirst && mx > 0.0f))) {
            k_exp = exponent(wave_max(mx), 8);
            kfirst = false;
        }
        if constexpr (PACKED) {
            const float by = __builtin_amdgcn_ldexpf(16.0f, -k_exp);
#pragma unroll
            for (int u = 0; u < DC; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ksc[u][e] *= by;
                    kzr[u][e] *= by;
                }
        }
    };
    auto k_token = [&](const int u, const int j, const uint32_t mask) {
        const int kc = 32 * u + 4 * kcq;
        float x[4];
        if constexpr (PACKED) {
            const uint32_t b = 0x0c0c0400u + 0x0101u * (ktq & 3);
            const uint32_t codes = __builtin_amdgcn_perm(kx[u][1], kx[u][0], b) | (__builtin_amdgcn_perm(kx[u][3], kx[u][2], b) << 16);
            uint32_t y = (codes >> (2 * j)) & 0x03030303u;
            asm("" : "+v"(y));  // (or every code is extracted by an instruction of its own)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(static_cast<float>((y >> (8 * e)) & 0xffu), ksc[u][e], kzr[u][e]);
        } else {
            const bool in = ((mask >> (4 * ktq + j)) & 1u) && kc < D;
            const float by = __builtin_amdgcn_ldexpf(16.0f, -k_exp);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = in ? __uint_as_float(kx[u][4 * j + e]) * by : 0.0f;
        }
        const uint2 p = parts(x[0], x[1]), q = parts(x[2], x[3]);
        char* d = lds + (4 * ktq + j) * L::KS + 2 * kc;
        *reinterpret_cast<uint2*>(d + L::KHI) = make_uint2(p.x, q.x);
        *reinterpret_cast<uint2*>(d + L::KLO) = make_uint2(p.y, q.y);
    };
    // V's exponent, likewise, and packed V's scales and zeros to LDS.
    auto ready_v = [&](const uint32_t mask) {
        float mx = 0.0f, x = 0.0f;
        const bool in = (mask >> n) & 1u;
        if constexpr (PACKED) {
            x = F16M ? half_lo(vm) : __uint_as_float(vm);
            mx = lane < 32 && in ? fabsf(x) : 0.0f;
        } else {
#pragma unroll
            for (int u = 0; u < DC; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    mx = fmaxf(mx, ((mask >> (4 * vtq + i / 4)) & 1u) && 32 * u + 4 * vcq < D ? fabsf(__uint_as_float(vx[u][i])) : 0.0f);
        }
        // (packed: a scale up to 2 2^v_exp stays in reach, P <= 2^14)
        const bool past = PACKED ? __builtin_amdgcn_ldexpf(mx, -v_exp) >= 2.0f : __builtin_amdgcn_ldexpf(mx, 4 - v_exp) >= kLimit;
        if (__ballot(past || (vfirst && mx > 0.0f))) {
            const int e = exponent(wave_max(mx), PACKED ? 0 : 8);
            const float f = __builtin_amdgcn_ldexpf(1.0f, v_exp - e);
            st.pz *= f;
#pragma unroll
            for (int s = 0; s < DC; ++s) acc[s] *= f;
            v_exp = e;
            vfirst = false;
        }
        if constexpr (PACKED) {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            const float y = lane < 32 ? x : __builtin_fmaf(1.5f, __uint_as_float(sw[0]), x);
            reinterpret_cast<float*>(lds + L::VMETA)[lane] = in ? __builtin_amdgcn_ldexpf(y, -v_exp) : 0.0f;
        }
    };
    auto v_channel = [&](const int u, const int k, const uint32_t mask) {
        const int vc = 32 * u + 4 * vcq;
        char* d = lds + (vc + k) * L::VS + 32 * (vtq >> 2) + 16 * (vtq & 1) + 8 * ((vtq >> 1) & 1);
        if constexpr (PACKED) {
            const uint32_t b = 0x0c040c00u + 0x00010001u * (vcq & 3), mk = 0x00060006u << (2 * k);
            const uint32_t y0 = __builtin_amdgcn_perm(vx[u][1], vx[u][0], b) << 1, y1 = __builtin_amdgcn_perm(vx[u][3], vx[u][2], b) << 1;
            const _Float16 c = static_cast<_Float16>(1024.0f + 3.0f * static_cast<float>(1 << (2 * k)));
            const mf_h2 off = {c, c};
            const mf_h2 z0 = __builtin_bit_cast(mf_h2, (y0 & mk) | 0x64006400u) - off;
            const mf_h2 z1 = __builtin_bit_cast(mf_h2, (y1 & mk) | 0x64006400u) - off;
            *reinterpret_cast<uint2*>(d + L::V) = make_uint2(__builtin_bit_cast(uint32_t, z0), __builtin_bit_cast(uint32_t, z1));
        } else {
            const float by = __builtin_amdgcn_ldexpf(16.0f, -v_exp);
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = ((mask >> (4 * vtq + j)) & 1u) && vc < D ? __uint_as_float(vx[u][4 * j + k]) * by : 0.0f;
            const uint2 p = parts(y[0], y[1]), q = parts(y[2], y[3]);
            *reinterpret_cast<uint2*>(d + L::V) = make_uint2(p.x, q.x);
            *reinterpret_cast<uint2*>(d + L::VLO) = make_uint2(p.y, q.y);
        }
    };

    fetch_k(t0);
    fetch_v(t0);
    const Row row = row_of(a, kvh, row0 + n, rows);
    mf_u4 qh[ST], ql[ST];
    const float crow = queries<ST>(a, row, h, neg1, qh, ql);
    uint32_t mask = mask_of(t0);
    ready_k(mask);
#pragma unroll
    for (int i = 0; i < 4 * DC; ++i) k_token(i / 4, i % 4, mask);
    fetch_k(min(t0 + 1, t1 - 1));
#pragma unroll 1
    for (int k = t0; k < t1; ++k) {
        ready_v(mask);
        wave_lds_sync();
        mf_f16 d;
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] = 0.0f;
        {
            const char* kl = lds + n * L::KS + 16 * h;
            mf_u4 kh[2], kw[2];
            auto load_k = [&](const int s) {
                kh[s & 1] = *reinterpret_cast<const mf_u4*>(kl + L::KHI + 32 * s);
                kw[s & 1] = *reinterpret_cast<const mf_u4*>(kl + L::KLO + 32 * s);
            };
            constexpr int PIECES = 4 * DC, SLOTS = 3 * ST;
            load_k(0);
            slot_end();
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                const int s = i / 3;
                if (i % 3 == 0 && s + 1 < ST) load_k(s + 1);
                d = mfma32x32x16(i % 3 == 2 ? kw[s & 1] : kh[s & 1], i % 3 == 0 ? ql[s] : qh[s], d);
#pragma unroll
                for (int o = i * PIECES / SLOTS; o < (i + 1) * PIECES / SLOTS; ++o) v_channel(o / 4, o % 4, mask);
                slot_end();
            }
        }
        fetch_v(min(k + 1, t1 - 1));
        wave_lds_sync();
        mf_u4 vh[2], vw[2], ph[2], pl[2];
        auto load_v = [&](const int s) {
            const char* x = lds + (32 * (s >> 1) + n) * L::VS + 32 * (s & 1) + 16 * h;
            vh[s & 1] = *reinterpret_cast<const mf_u4*>(x + L::V);
            if constexpr (!PACKED) vw[s & 1] = *reinterpret_cast<const mf_u4*>(x + L::VLO);
        };
        softmax32<DC, PACKED>(st, d, acc, mask, __builtin_amdgcn_ldexpf(crow, k_exp), lds + L::VMETA, lane, neg1, ph, pl,
                              [&]() { load_v(0); });
        mask = mask_of(min(k + 1, t1 - 1));
        ready_k(mask);
        constexpr int PR = PACKED ? 2 : 3, SLOTS = 2 * DC * PR, PIECES = 4 * DC;
        slot_end();
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int s = i / PR, q = i % PR;
            if (q == 0 && s + 1 < 2 * DC) load_v(s + 1);
            acc[s >> 1] = mfma32x32x16(q == 0 ? pl[s & 1] : ph[s & 1], !PACKED && q == 1 ? vw[s & 1] : vh[s & 1], acc[s >> 1]);
#pragma unroll
            for (int o = i * PIECES / SLOTS; o < (i + 1) * PIECES / SLOTS; ++o) k_token(o / 4, o % 4, mask);
            slot_end();
        }
        fetch_k(min(k + 2, t1 - 1));
        wave_lds_sync();
    }
    store32<DC, 4, PACKED>(a, row, st, acc, v_exp, lane, row0, rows, slot);
}

// The same for head dims above 128, whose accumulators leave registers for 16 rows per wave. Eight waves,
// on the same tile with rows of their own.
//
// The loop is a pipeline over the tiles: while the matrix cores multiply Q with
// K of tile k, the VALU turns tile k - 1's logits into P; while they multiply P
// with V of tile k - 1, it stages K of tile k + 1 and V of tile k, whose loads
// went out at the top. One barrier per tile.
template <bool PACKED, typename MetaT>
__device__ __forceinline__ void wide_body(const SharedArgs& a, char* lds, const Tiers& t, const int kvh,
                                            const int row0, const int rows, const int t0, const int t1,
                                            const int slot) {
    constexpr int DC = kWideDC, WM = 8;
    using L = TileLds<DC>;
    constexpr bool F16M = sizeof(MetaT) == 2;
    float neg1 = -1.0f;
    asm("" : "+s"(neg1));
    auto parts = [&](const float x0, const float x1) { return tt::parts(x0, x1, neg1); };
    const int lane = threadIdx.x & 63;
    const int wave = scalar(static_cast<int>(threadIdx.x) >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int G = a.Hq / a.Hkv;
    const int D = a.D;
    const size_t Hkv = static_cast<size_t>(a.Hkv);
    // A unit is 64 lanes x (4 tokens x 4 channels) of a tile: 32 channels. Each wave stages one of K and one of V.
    static_assert(WM == DC, "");
    // K units: lane = (token quad, channel quad); V units the other way round,
    // so that the writes of V's transposed rows spread over the banks.
    const int ktq = lane >> 3, kcq = lane & 7;
    const int vtq = lane & 7, vcq = lane >> 3;
    const int kc = 32 * wave + 4 * kcq, vc = 32 * wave + 4 * vcq;  // first channels
    const int kt0 = 4 * ktq;                                       // first token
    const bool has_meta = wave == 0;                               // stages V's scales and zeros

    // The tile in flight, as it lies in memory.
    mf_u4 kx[PACKED ? 3 : 4];               // packed: words, scale, zero; FP32: tokens
    uint32_t vx[4][PACKED ? 1 : 4];         // packed: words of 4 tokens; FP32: 4 tokens' channels
    uint2 idv = make_uint2(0u, 0u);
    uint32_t vm = 0u;                        // packed: V scale (lanes 0-31) or zero (lanes 32-63) of token lane % 32
    auto fetch_k = [&](const int tile) {
        const int s0 = kTile * tile;
        const int c = min(kc, D - 4);
        if constexpr (PACKED) {
            const int last = t.slots - 1;
            idv = *reinterpret_cast<const uint2*>(t.ids + min(s0 + (lane & 31), last));
            const int s = min(s0 + 4 * ktq, last);
            const size_t km = static_cast<size_t>(a.kgs == 32 ? s >> 5 : s >> 4) * Hkv * D + c;
            kx[0] = *reinterpret_cast<const un_u4*>(t.kp + static_cast<size_t>(s >> 4) * Hkv * D + c);
            if constexpr (!F16M) {
                kx[1] = *reinterpret_cast<const un_u4*>(t.ks + 4 * km);
                kx[2] = *reinterpret_cast<const un_u4*>(t.kz + 4 * km);
            } else {
                const un_u2 ps = *reinterpret_cast<const un_u2*>(t.ks + 2 * km);
                const un_u2 pz = *reinterpret_cast<const un_u2*>(t.kz + 2 * km);
                kx[1] = mf_u4{ps[0], ps[1], pz[0], pz[1]};
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                kx[j] = *reinterpret_cast<const un_u4*>(t.dk + min(s0 + kt0 + j, t.nd - 1) * Hkv * D + c);
        }
    };
    auto fetch_v = [&](const int tile) {
        const int s0 = kTile * tile;
        const int c = min(vc, D - 4);
        if constexpr (PACKED) {
            const int last = t.slots - 1;
            if (has_meta) {
                const size_t at = min(s0 + (lane & 31), last) * Hkv * sizeof(MetaT);
                vm = *reinterpret_cast<const MetaBits<MetaT>*>((lane < 32 ? t.vs : t.vz) + at);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                vx[j][0] = t.vp[static_cast<size_t>(min(s0 + 4 * vtq + j, last)) * Hkv * (D / 16) + (c >> 4)];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const un_u4 y = *reinterpret_cast<const un_u4*>(t.dv + min(s0 + 4 * vtq + j, t.nd - 1) * Hkv * D + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) vx[j][e] = y[e];
            }
        }
    };
    // Bit j: token j of the tile is attended (packed: of the K tile in flight).
    auto mask_of = [&](const int tile) -> uint32_t {
        const int left = (PACKED ? t.slots : t.nd) - kTile * tile;
        const uint32_t in = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
        if constexpr (PACKED) return static_cast<uint32_t>(__ballot((idv.x & idv.y) != 0xffffffffu)) & in;
        return in;
    };

    float* peak = reinterpret_cast<float*>(lds + 2 * L::BYTES);  // [tile's parity][key, value]
    // A tile's largest key or value where it asks for another scale: too large for f16 at this one, or (first) any.
    // The peaks only grow and so do the exponents after the first: none is ever cleared.
    // Positive floats order like their bits. (An infinity has no scale that helps: it is left to make NaN of what
    // reads it.)
    auto report = [&](const float x, const float back, const bool first, float* to) {
        const bool tell = x >= kLimit || (first && x > 0.0f);
        if (__ballot(tell))
            if (tell && x < __builtin_huge_valf()) atomicMax(reinterpret_cast<int*>(to), __float_as_int(fminf(x * back, 3.0e38f)));
    };

    // f16 parts of the fetched K (scaled by 2^(4 - ke)).
    auto stage_k = [&](char* tl, const uint32_t mask, const int ke) -> float {
        const float ksc = __builtin_amdgcn_ldexpf(16.0f, -ke);
        float mx = 0.0f;
        float x[4][4];  // [token][channel]
        if constexpr (PACKED) {
            // no attended token: the block's scale and zero may be anything
            const bool any = ((mask >> (4 * ktq)) & 15u) != 0u && kc < D;
            float sc[4], zr[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (F16M) {
                    const uint32_t hs = kx[1][e >> 1], hz = kx[1][2 + (e >> 1)];
                    sc[e] = (e & 1) ? half_hi(hs) : half_lo(hs);
                    zr[e] = (e & 1) ? half_hi(hz) : half_lo(hz);
                } else {
                    sc[e] = __uint_as_float(kx[1][e]);
                    zr[e] = __uint_as_float(kx[2][e]);
                }
                sc[e] = any ? sc[e] * ksc : 0.0f;
                zr[e] = any ? zr[e] * ksc : 0.0f;
                mx = fmaxf(mx, fmaxf(fabsf(zr[e]), fabsf(__builtin_fmaf(3.0f, sc[e], zr[e]))));
            }
            // the quad's codes, one byte per channel, then one code per byte
            const uint32_t b = 0x0c0c0400u + 0x0101u * (ktq & 3);
            const uint32_t lo = __builtin_amdgcn_perm(kx[0][1], kx[0][0], b);
            const uint32_t hi = __builtin_amdgcn_perm(kx[0][3], kx[0][2], b);
            const uint32_t w = lo | (hi << 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t y = (w >> (2 * j)) & 0x03030303u;
                asm("" : "+v"(y));  // (or every code is extracted by an instruction of its own)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[j][e] = __builtin_fmaf(static_cast<float>((y >> (8 * e)) & 0xffu), sc[e], zr[e]);
            }
        } else {
            const uint32_t mine = mask >> kt0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[j][e] = ((mine >> j) & 1u) && kc < D ? __uint_as_float(kx[j][e]) * ksc : 0.0f;
                    mx = fmaxf(mx, fabsf(x[j][e]));
                }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint2 p = parts(x[j][0], x[j][1]), q = parts(x[j][2], x[j][3]);
            char* d = tl + (kt0 + j) * L::KS + 2 * kc;
            *reinterpret_cast<uint2*>(d + L::KHI) = make_uint2(p.x, q.x);
            *reinterpret_cast<uint2*>(d + L::KLO) = make_uint2(p.y, q.y);
        }
        return mx;
    };
    // Packed: the centred codes (2 q - 3) 4^(c % 4), exact, of channels c. FP32: f16 parts of V 2^(4 - ve). Token quad vtq
    // sits in the MFMA order: 8 tokens per lane group, its half by the 16-token tile.
    auto stage_v = [&](char* tl, const uint32_t mask, const int ve) -> float {
        float mx = 0.0f;
        char* d = tl + vc * L::VS + 16 * (vtq & 3) + 8 * (vtq >> 2);
        if constexpr (PACKED) {
            // channels past head_dim hold codes of others, in columns that are not stored
            const uint32_t b = 0x0c040c00u + 0x00010001u * (vcq & 3);
            // the codes of the lane's first channel at bit 1 of each half
            const uint32_t y0 = __builtin_amdgcn_perm(vx[1][0], vx[0][0], b) << 1;
            const uint32_t y1 = __builtin_amdgcn_perm(vx[3][0], vx[2][0], b) << 1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const _Float16 c = static_cast<_Float16>(1024.0f + 3.0f * static_cast<float>(1 << (2 * k)));
                const mf_h2 off = {c, c};
                const uint32_t mk = 0x00060006u << (2 * k);
                const mf_h2 z0 = __builtin_bit_cast(mf_h2, (y0 & mk) | 0x64006400u) - off;
                const mf_h2 z1 = __builtin_bit_cast(mf_h2, (y1 & mk) | 0x64006400u) - off;
                *reinterpret_cast<uint2*>(d + k * L::VS + L::V) =
                    make_uint2(__builtin_bit_cast(uint32_t, z0), __builtin_bit_cast(uint32_t, z1));
            }
        } else {
            const float vsc = __builtin_amdgcn_ldexpf(16.0f, -ve);
            const uint32_t mine = (mask >> (4 * vtq)) & 15u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = ((mine >> j) & 1u) && vc < D ? __uint_as_float(vx[j][e]) * vsc : 0.0f;
                    mx = fmaxf(mx, fabsf(y[j]));
                }
                const uint2 p = parts(y[0], y[1]), q = parts(y[2], y[3]);
                *reinterpret_cast<uint2*>(d + e * L::VS + L::V) = make_uint2(p.x, q.x);
                *reinterpret_cast<uint2*>(d + e * L::VS + L::VLO) = make_uint2(p.y, q.y);
            }
        }
        return mx;
    };
    // Packed: V's scale 2^-ve and the zero of the centred codes, vz + 1.5 vs, of the tile's tokens, zeros where masked.
    auto stage_meta = [&](char* tl, const uint32_t mask, const int ve) -> float {
        const float x = F16M ? half_lo(vm) : __uint_as_float(vm);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        float y = lane < 32 ? x : __builtin_fmaf(1.5f, __uint_as_float(sw[0]), x);
        y = ((mask >> (lane & 31)) & 1u) ? __builtin_amdgcn_ldexpf(y, -ve) : 0.0f;
        reinterpret_cast<float*>(tl + L::VMETA)[lane] = y;
        return lane < 32 ? fabsf(y) : 0.0f;
    };

    fetch_k(t0);
    fetch_v(t0);
    float2 top;  // the first tile's largest key and value
    {
        const uint32_t m = mask_of(t0);
        float kmx = 0.0f, vmx = 0.0f;
        if constexpr (PACKED) {
            const bool any = ((m >> (4 * ktq)) & 15u) != 0u && kc < D;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t hs = kx[1][F16M ? e >> 1 : e], hz = kx[F16M ? 1 : 2][F16M ? 2 + (e >> 1) : e];
                const float sc = F16M ? ((e & 1) ? half_hi(hs) : half_lo(hs)) : __uint_as_float(hs);
                const float zr = F16M ? ((e & 1) ? half_hi(hz) : half_lo(hz)) : __uint_as_float(hz);
                if (any) kmx = fmaxf(kmx, fmaxf(fabsf(zr), fabsf(__builtin_fmaf(3.0f, sc, zr))));
            }
            if (has_meta && lane < 32 && ((m >> lane) & 1u)) vmx = fabsf(F16M ? half_lo(vm) : __uint_as_float(vm));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (((m >> (kt0 + j)) & 1u) && kc < D) kmx = fmaxf(kmx, fabsf(__uint_as_float(kx[j][e])));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (((m >> (4 * vtq + j)) & 1u) && vc < D) vmx = fmaxf(vmx, fabsf(__uint_as_float(vx[j][e])));
        }
        top = group_max<WM>(kmx, vmx, lds, wave, lane);
    }

    // Q' = Q 2^(12 - e), e the exponent of the row's largest value, as the QK B operand: row n, channels 32 s + 8 g .. + 7.
    const bool rowed = row0 + 16 * wave < rows;  // a wave without rows multiplies nothing (P = 0)
    mf_u4 qh[DC], ql[DC];
    float crow;  // log2 units per unit of the product
    {
        const int r = row0 + 16 * wave + n;
        const bool live = r < rows;
        const int seq = live ? r / G : 0;
        const int h = kvh * G + (live ? r % G : 0);
        const float* q = global_ptr(a.seqs[seq].Q) + static_cast<size_t>(h) * D;
        un_u4 x[DC][2];
#pragma unroll
        for (int s = 0; s < DC; ++s) {
            const int c = min(32 * s + 8 * g, D - 8);
            x[s][0] = *reinterpret_cast<const un_u4*>(q + c);
            x[s][1] = *reinterpret_cast<const un_u4*>(q + c + 4);
        }
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < DC; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (!live || 32 * s + 8 * g >= D) x[s][j >> 2][j & 3] = 0u;
                mx = fmaxf(mx, fabsf(__uint_as_float(x[s][j >> 2][j & 3])));
            }
        mx = xrow_max(mx);
        const int e = (mx > 0.0f) ? __builtin_amdgcn_frexp_expf(mx) : 0;
#pragma unroll
        for (int s = 0; s < DC; ++s) {
            uint2 p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                p[j] = parts(__builtin_amdgcn_ldexpf(__uint_as_float(x[s][j >> 1][2 * (j & 1)]), 12 - e),
                             __builtin_amdgcn_ldexpf(__uint_as_float(x[s][j >> 1][2 * (j & 1) + 1]), 12 - e));
            qh[s] = mf_u4{p[0].x, p[1].x, p[2].x, p[3].x};
            ql[s] = mf_u4{p[0].y, p[1].y, p[2].y, p[3].y};
        }
        crow = __builtin_amdgcn_ldexpf(a.scale2, e - 16);
    }

    mf_f4 acc[2 * DC], d[2];
    mf_u4 ph, pl;
    float mr = -3.0e38f, l = 0.0f, pz = 0.0f;
    ph = pl = mf_u4{0u, 0u, 0u, 0u};
    d[0] = d[1] = mf_f4{kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
    for (int s = 0; s < 2 * DC; ++s) acc[s] = mf_f4{0.0f, 0.0f, 0.0f, 0.0f};
    // Exponents of the scales of K and V (uniform over the workgroup), and whether no tile has set them yet; that of
    // the K behind the logits in d.
    int k_exp = exponent(top.x, 8), v_exp = exponent(top.y, PACKED ? 0 : 8), d_exp = 0;
    bool kfirst = !__ballot(top.x > 0.0f), vfirst = !__ballot(top.y > 0.0f);
    lds_barrier();
    if (threadIdx.x < 4) peak[threadIdx.x] = 0.0f;
    // The start multiplies P = 0 with what this buffer holds.
    for (int x = 16 * threadIdx.x; x < 2 * 32 * DC * L::VS; x += 16 * 64 * WM)
        *reinterpret_cast<mf_u4*>(lds + ((t0 - 1) & 1) * L::BYTES + L::V + x) = mf_u4{0u, 0u, 0u, 0u};

    // At the top of the loop K of tile k and V of tile k - 1 are staged. `again`: they have to be, at the start or
    // with other exponents; nothing is multiplied then (P is zero).
    int again = 1;
    asm("" : "+s"(again));  // (or the compiler makes a loop of its own of the start)
    uint32_t m0 = 0u, m1 = 0u;  // masks of tiles k - 1 and k
    int k = t0;
    bool more;
#pragma unroll 1
    do {
        lds_barrier();
        if (!again || k > t0 || m1) {
            const float2 pk = *reinterpret_cast<const float2*>(peak + 2 * (k & 1));
            const float pv_ = peak[2 * ((k - 1) & 1) + 1];
            int kn = k_exp, vn = v_exp;
            if (__ballot(pk.x > 0.0f)) {
                const int e = exponent(pk.x, 8);  // (a peak past the limit asks for 4 more at least)
                if (e - 3 > k_exp || kfirst) kn = e;
                kfirst = false;
            }
            if (__ballot(pv_ > 0.0f)) {
                const int e = exponent(pv_, PACKED ? 0 : 8);
                if (e - (PACKED ? 1 : 3) > v_exp || vfirst) vn = e;
                vfirst = false;
            }
            again = kn != k_exp || vn != v_exp ? 1 : 0;
            if (again) {
                const float f = __builtin_amdgcn_ldexpf(1.0f, v_exp - vn);
                pz *= f;
                ph = pl = mf_u4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int s = 0; s < 2 * DC; ++s) acc[s] *= f;
                k_exp = kn;
                v_exp = vn;
                lds_barrier();
            }
        }
        const int kt = min(again ? k : k + 1, t1 - 1), vt = max(min(again ? k - 1 : k, t1 - 1), t0);
        fetch_k(kt);
        fetch_v(vt);
        const char* kl = lds + (k & 1) * L::BYTES;
        char* vl = lds + ((k - 1) & 1) * L::BYTES;
        if (rowed && !again) {
            // Softmax of tile k - 1's logits, P (packed: P times V's scale) as the PV A operand; QK of tile k.
            if (m0 != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool in = (m0 >> (16 * i + 4 * g + r)) & 1u;
                        d[i][r] = in ? d[i][r] : kNegInf;
                    }
            }
            const float c = __builtin_amdgcn_ldexpf(crow, d_exp);
            float mx = max3(max3(d[0][0], d[0][1], d[0][2]), d[0][3], d[1][0]);
            mx = max3(mx, max3(d[1][1], d[1][2], d[1][3]), mx);
            mx = __builtin_fmaf(mx, c, -kUp);
            // the reference moves only when a row's maximum passes it by more than the slack
            if (__ballot(mx > mr + kSlack)) {
                mx = xrow_max(mx);
                const bool up = mx > mr + kSlack;
                const float mn = up ? mx : mr;
                const float al = up ? __builtin_amdgcn_exp2f(mr - mn) : 1.0f;
                l *= al;
                pz *= al;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float ar = __shfl(al, 4 * g + r, 64);
#pragma unroll
                    for (int q = 0; q < 2 * DC; ++q) acc[q][r] *= ar;
                }
                mr = mn;
            }
            mf_f4 dn[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) dn[i] = mf_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < DC; ++s) {
                mf_u4 kh[2], kw[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const char* p = kl + (16 * i + n) * L::KS + 64 * s + 16 * g;
                    kh[i] = *reinterpret_cast<const mf_u4*>(p + L::KHI);
                    kw[i] = *reinterpret_cast<const mf_u4*>(p + L::KLO);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) dn[i] = mfma16x16x32(kh[i], ql[s], dn[i]);
#pragma unroll
                for (int i = 0; i < 2; ++i) dn[i] = mfma16x16x32(kw[i], qh[s], dn[i]);
#pragma unroll
                for (int i = 0; i < 2; ++i) dn[i] = mfma16x16x32(kh[i], qh[s], dn[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                mf_f4 vs, vz;
                if constexpr (PACKED) {
                    vs = *reinterpret_cast<const mf_f4*>(vl + L::VMETA + 64 * i + 16 * g);
                    vz = *reinterpret_cast<const mf_f4*>(vl + L::VMETA + 128 + 64 * i + 16 * g);
                }
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(d[i][r], c, -mr));
                    l += p[r];
                    if constexpr (PACKED) {
                        pz = __builtin_fmaf(p[r], vz[r], pz);
                        p[r] *= vs[r];
                    }
                }
                const uint2 x = parts(p[0], p[1]), y = parts(p[2], p[3]);
                ph[2 * i] = x.x;
                ph[2 * i + 1] = y.x;
                pl[2 * i] = x.y;
                pl[2 * i + 1] = y.y;
                d[i] = dn[i];
            }
            interleave<6 * DC>();
            d_exp = k_exp;
        }
        // PV of tile k - 1, and the fetched tiles to LDS.
#pragma unroll
        for (int q = 0; q < 2 * DC; ++q) {
            const char* p = vl + (16 * q + n) * L::VS + 16 * g;
            const mf_u4 vh = *reinterpret_cast<const mf_u4*>(p + L::V);
            acc[q] = mfma16x16x32(pl, vh, acc[q]);
            if constexpr (!PACKED) {
                const mf_u4 vw = *reinterpret_cast<const mf_u4*>(p + L::VLO);
                acc[q] = mfma16x16x32(ph, vw, acc[q]);
            }
            acc[q] = mfma16x16x32(ph, vh, acc[q]);
        }
        const uint32_t mk = mask_of(kt);
        const uint32_t mv = vt == kt ? mk : (vt == k ? m1 : m0);
        const int kb = again ? k & 1 : (k + 1) & 1, vb = again ? (k - 1) & 1 : k & 1;
        const float kmx = stage_k(lds + kb * L::BYTES, mk, k_exp);
        const float vmx = stage_v(lds + vb * L::BYTES, mv, v_exp);
        interleave<2 * DC * (PACKED ? 2 : 3)>();
        report(kmx, __builtin_amdgcn_ldexpf(0.0625f, k_exp), kfirst, peak + 2 * kb);
        if constexpr (!PACKED)
            report(vmx, __builtin_amdgcn_ldexpf(0.0625f, v_exp), vfirst, peak + 2 * vb + 1);
        if constexpr (PACKED) {
            // a scale up to 2 2^v_exp stays in reach (P <= 2^14): reported in units of kLimit / 2
            if (has_meta)
                report(stage_meta(lds + vb * L::BYTES, mv, v_exp) * (0.5f * kLimit),
                       __builtin_amdgcn_ldexpf(2.0f / kLimit, v_exp), vfirst, peak + 2 * vb + 1);
        }
        if (!again) m0 = m1;
        m1 = mk;
        more = again || k != t1;
        k += again ? 0 : 1;
        again = 0;
    } while (more);

    // The partial in units of V: acc holds 16 V 2^-v_exp (FP32 tiles), or 2 4^(c % 4) of it without the centred zero.
    l = xrow_sum(l);
    const float back = __builtin_amdgcn_ldexpf(1.0f, v_exp - (PACKED ? 1 + 2 * (n & 3) : 4));
    const float z = PACKED ? __builtin_amdgcn_ldexpf(xrow_sum(pz), v_exp) : 0.0f;
    const int rn = row0 + 16 * wave + n;
    // row rn's partial, behind its sequence's own slots
    const int seq = rn < rows ? rn / G : 0;
    const int ns = a.slot_base[seq + 1] - a.slot_base[seq];
    const int h = kvh * G + (rn < rows ? rn % G : 0);
    const uint32_t pi = static_cast<uint32_t>(a.slot_base[seq] * a.Hq + h * ns + (ns - a.prefix_slots + slot));
    if (g == 0 && rn < rows) {
        a.ml[2 * static_cast<size_t>(pi)] = l > 0.0f ? mr : kNegInf;
        a.ml[2 * static_cast<size_t>(pi) + 1] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float zr = PACKED ? __shfl(z, 4 * g + r, 64) : 0.0f;
        const uint32_t pr = static_cast<uint32_t>(__shfl(static_cast<int>(pi), 4 * g + r, 64));
        if (row0 + 16 * wave + 4 * g + r >= rows) continue;
        float* o = a.acc + static_cast<size_t>(pr) * D + n;
#pragma unroll
        for (int q = 0; q < 2 * DC; ++q)
            if (16 * q < D) o[16 * q] = __builtin_fmaf(acc[q][r], back, zr);
    }
}

// First of `count` items of part i of `parts`.
__device__ __forceinline__ int share(const int count, const int i, const int parts) {
    return scalar(static_cast<int>(static_cast<long long>(count) * i / parts));
}

// Grid: slots x (KV heads x row chunks); slot s of all heads and chunks on XCD
// s % 8, back to back, so that a tile's lines come from memory once. Slots
// [0, packed_slots) share the packed tiles, the others the FP32 ones.
template <int DC, int WM, bool PACKED, typename MetaT>
__device__ __forceinline__ void any_body(const SharedArgs& a, char* lds, const Tiers& t, const int kvh, const int row0,
                                         const int rows, const int t0, const int t1, const int slot) {
    if constexpr (DC > 4)
        wide_body<PACKED, MetaT>(a, lds, t, kvh, row0, rows, t0, t1, slot);
    else
        shared_body<DC, WM, PACKED, MetaT>(a, lds, t, kvh, row0, rows, t0, t1, slot);
}

template <int DC, int WM, typename MetaT>
__global__ void __launch_bounds__(64 * WM) __attribute__((amdgpu_waves_per_eu(Config<DC, WM>::PER_EU)))
attn_shared_kernel(const SharedArgs a) {
    __shared__ __align__(16) char lds[Config<DC, WM>::LDS];
    const unsigned id = blockIdx.x;
    const unsigned q = id >> 3;
    const unsigned hc = static_cast<unsigned>(a.Hkv * a.chunks);
    const int hz = static_cast<int>(q % hc);
    const int s = static_cast<int>((q / hc) * 8 + (id & 7));
    if (s >= a.prefix_slots) return;
    const int kvh = hz / a.chunks, chunk = hz - kvh * a.chunks;
    const int rows = a.nseq * (a.Hq / a.Hkv), row0 = chunk * Config<DC, WM>::ROWS;
    const Tiers t = tiers_of(a, kvh);
    if (s < a.packed_slots) {
        const int tiles = (t.slots + kTile - 1) / kTile;
        any_body<DC, WM, true, MetaT>(a, lds, t, kvh, row0, rows, share(tiles, s, a.packed_slots),
                                      share(tiles, s + 1, a.packed_slots), s);
    } else {
        const int tiles = (t.nd + kTile - 1) / kTile, nd = a.prefix_slots - a.packed_slots;
        any_body<DC, WM, false, MetaT>(a, lds, t, kvh, row0, rows, share(tiles, s - a.packed_slots, nd),
                                       share(tiles, s - a.packed_slots + 1, nd), s);
    }
}

// Waves with tiles of their own: four slots to a workgroup, those of all heads and chunks back to back on one XCD.
template <int DC>
struct Lone {
    static constexpr int ROWS = kLoneRows;
    static constexpr int LDS = 4 * TileLds<DC>::BYTES;
};
template <int DC, typename MetaT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) attn_shared_few_kernel(const SharedArgs a) {
    __shared__ __align__(16) char lds[Lone<DC>::LDS];
    const unsigned id = blockIdx.x;
    const unsigned q = id >> 3;
    const unsigned hc = static_cast<unsigned>(a.Hkv * a.chunks);
    const int hz = static_cast<int>(q % hc);
    const int wave = scalar(static_cast<int>(threadIdx.x) >> 6);
    const int s = 4 * static_cast<int>((q / hc) * 8 + (id & 7)) + wave;
    if (s >= a.prefix_slots) return;
    const int kvh = hz / a.chunks, chunk = hz - kvh * a.chunks;
    const int rows = a.nseq * (a.Hq / a.Hkv), row0 = chunk * Lone<DC>::ROWS;
    const Tiers t = tiers_of(a, kvh);
    char* own = lds + wave * TileLds<DC>::BYTES;
    if (s < a.packed_slots) {
        const int tiles = (t.slots + kTile - 1) / kTile;
        lone_body<DC, true, MetaT>(a, own, t, kvh, row0, rows, share(tiles, s, a.packed_slots), share(tiles, s + 1, a.packed_slots), s);
    } else {
        const int tiles = (t.nd + kTile - 1) / kTile, nd = a.prefix_slots - a.packed_slots;
        lone_body<DC, false, MetaT>(a, own, t, kvh, row0, rows, share(tiles, s - a.packed_slots, nd),
                                    share(tiles, s - a.packed_slots + 1, nd), s);
    }
}

template <int DC>
int launch_few(SharedArgs a, const int rows, hipStream_t st) {
    a.chunks = (rows + Lone<DC>::ROWS - 1) / Lone<DC>::ROWS;
    const long long wgs = static_cast<long long>((a.prefix_slots + 31) / 32) * 8 * a.Hkv * a.chunks;
    if (wgs > 0x00ffffffLL) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "attention grid too large");
    const dim3 grid(static_cast<unsigned>(wgs));
    if (a.meta_fp16)
        hipLaunchKernelGGL((attn_shared_few_kernel<DC, uint16_t>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((attn_shared_few_kernel<DC, float>), grid, dim3(256), 0, st, a);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

template <int DC, int WM>
int launch(SharedArgs a, const int rows, hipStream_t st) {
    a.chunks = (rows + Config<DC, WM>::ROWS - 1) / Config<DC, WM>::ROWS;
    const long long wgs = static_cast<long long>((a.prefix_slots + 7) / 8) * 8 * a.Hkv * a.chunks;
    if (wgs > 0x00ffffffLL) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "attention grid too large");
    const dim3 grid(static_cast<unsigned>(wgs));
    if (a.meta_fp16)
        hipLaunchKernelGGL((attn_shared_kernel<DC, WM, uint16_t>), grid, dim3(64 * WM), 0, st, a);
    else
        hipLaunchKernelGGL((attn_shared_kernel<DC, WM, float>), grid, dim3(64 * WM), 0, st, a);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

// The instantiation that serves `rows` rows per KV head: 32-channel chunks DC, and four waves or, past their rows, eight.
template <int DC, typename F>
auto for_rows(const int rows, F&& f) {
    using C = std::integral_constant<int, DC>;
    if constexpr (DC > 4) {
        return f(C{}, std::integral_constant<int, 8>{});
    } else {
        if (rows <= 128) return f(C{}, std::integral_constant<int, 4>{});
        return f(C{}, std::integral_constant<int, 8>{});
    }
}
template <typename F>
auto for_shape(const int D, const int rows, F&& f) {
    if (D <= 64) return for_rows<2>(rows, f);
    if (D <= 96) return for_rows<3>(rows, f);
    if (D <= 128) return for_rows<4>(rows, f);
    return for_rows<kWideDC>(rows, f);
}

// The rows of a share of tiles, and the shares that a CU holds at a time.
struct Shape {
    int rows, per_cu;
};
Shape shape_of(const int D, const int rows, const bool lone) {
    if (lone) return Shape{kLoneRows, 4};
    return for_shape(D, rows, [&](auto dc, auto wm) {
        using C = Config<dc.value, wm.value>;
        return Shape{C::ROWS, C::PER_CU};
    });
}

}  // namespace

SharedPlan shared_plan(const tt_decode_seq& prefix, const tt_decode_seq* seqs, int nseq, int Hq, int Hkv, int D, int kgs,
                       int meta_fp16) {
    SharedPlan p;
    BatchPlan& b = p.batch;
    const int rows = nseq * (Hq / Hkv);
    const long long dense = (static_cast<long long>(prefix.dense_count) + kTile - 1) / kTile;
    const long long packed = (static_cast<long long>(prefix.num_blocks) * kgs + kTile - 1) / kTile;
    const long long tokens = static_cast<long long>(prefix.dense_count) + static_cast<long long>(prefix.num_blocks) * kgs;
    const double cost = packed + kDenseCost * dense;
    p.lone = D <= 128 && rows <= kLoneRows && cost * Hkv >= 256 * kLoneTiles;
    const Shape sh = shape_of(D, rows, p.lone);
    // One round of workgroups, each kind's share by what its tiles cost; fewer where another one's partials cost the merge
    // more than it saves the others in tiles (32 sequences behind 2k, 32/8 heads of 128: 41.9 -> 37.0 us).
    const long long groups = static_cast<long long>(Hkv) * ((rows + sh.rows - 1) / sh.rows);
    const double merge = 8.0 * nseq * Hq * D / kMergeRate;  // us per slot
    const double best = std::sqrt(tile_us(D) * cost / merge);
    long long slots = std::min<long long>(256LL * sh.per_cu / groups, std::llround(best));
    if (p.lone) slots = std::min<long long>(slots, std::llround(cost / 4));
    slots = std::max<long long>(1, slots);
    const double shared_us = kSharedUs + D / 16.0 + tile_us(D) * std::ceil(cost / slots) + merge * slots;
    p.per_seq = tokens > 0 && nseq <= kMaxBatchSeqs / 2 && walk_us(nseq, static_cast<double>(tokens), Hq, Hkv, D) <= shared_us ? 2 : 1;
    tt_decode_seq entries[kMaxBatchSeqs];
    for (int i = 0; i < nseq; ++i) {
        entries[p.per_seq * i] = seqs[i];
        if (p.per_seq == 2) {
            entries[2 * i + 1] = prefix;
            entries[2 * i + 1].mean_attn_weights = nullptr;
        }
    }
    p.entries = own_plan(entries, p.per_seq * nseq, p.per_seq, Hq, Hkv, D, kgs, meta_fp16);
    if (p.per_seq == 1 && tokens > 0) {
        long long np = packed ? std::max<long long>(1, std::llround(slots * packed / cost)) : 0;
        np = std::min(np, packed);
        long long nd = dense ? std::max<long long>(1, slots - np) : 0;
        nd = std::min(nd, dense);
        p.packed_slots = static_cast<int>(np);
        p.prefix_slots = static_cast<int>(np + nd);
    }
    b.nseq = nseq;
    for (int i = 0; i < nseq; ++i)
        b.slot_base[i + 1] = b.slot_base[i] + p.prefix_slots + p.entries.slot_base[p.per_seq * (i + 1)] -
                             p.entries.slot_base[p.per_seq * i];
    batch_layout(b, seqs, Hq, D, kgs);
    return p;
}

int shared_launch(const SharedPlan& plan, const tt_decode_seq& prefix, const tt_decode_seq* seqs_dev, int Hq, int Hkv,
                  int D, int kgs, int meta_fp16, void* ws, hipStream_t stream) {
    const BatchPlan& b = plan.batch;
    char* base = static_cast<char*>(ws);
    if (plan.prefix_slots > 0) {
        SharedArgs a;
        a.seqs = seqs_dev;
        a.prefix = prefix;
        a.ml = reinterpret_cast<float*>(base + b.off_ml);
        a.acc = reinterpret_cast<float*>(base + b.off_acc);
        a.scale2 = kLog2e / sqrtf(static_cast<float>(D));
        a.nseq = b.nseq;
        a.Hq = Hq;
        a.Hkv = Hkv;
        a.D = D;
        a.kgs = kgs;
        a.meta_fp16 = meta_fp16 ? 1 : 0;
        a.prefix_slots = plan.prefix_slots;
        a.packed_slots = plan.packed_slots;
        a.chunks = 1;
        std::memcpy(a.slot_base, b.slot_base, sizeof(a.slot_base));
        const int rows = b.nseq * (Hq / Hkv);
        const int rc = for_shape(D, rows, [&](auto dc, auto wm) {
            if constexpr (dc.value <= 4)
                if (plan.lone) return launch_few<dc.value>(a, rows, stream);
            return launch<dc.value, wm.value>(a, rows, stream);
        });
        if (rc) return rc;
    }
    const int rc = own_launch(plan, prefix, seqs_dev, Hq, Hkv, D, kgs, meta_fp16, ws, stream);
    if (rc) return rc;
    return batch_finalize(b, seqs_dev, Hq, D, kgs, ws, stream, true);
}

}  // namespace tt
