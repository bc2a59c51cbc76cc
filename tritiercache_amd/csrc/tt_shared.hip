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
//   QK  A = K (16 tokens x 32 channels), B = Q (32 channels x 16 rows):
//       lane (g = lane / 16, n = lane % 16) receives tokens 4 g .. 4 g + 3 of row n.
//   PV  A = P (16 rows x 32 tokens), B = V (32 tokens x 16 channels): the two
//       16-token QK results of a lane are its A operand as they lie, in the
//       token order k = 8 g + j <-> token 4 g + j (j < 4), 16 + 4 g + j - 4
//       (else), which V has in LDS.
// f16 covers 2^-14 .. 2^16 with all its bits, so the parts are scaled by
// powers of two: Q by its row's largest value (to below 2^12), K and V by 16 and,
// where a tile holds larger values than 4080 or the first one only values below
// 1/8, by the exponent that brings them back (k_exp, v_exp; the tile is staged
// again), P by the running reference m = max - 12 (P <= 2^14 with the slack of
// the lazy rescale).
#include "tt_shared.h"
#include "tt_wave.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tt {
namespace {

// Attended tokens of all sequences together (the prefix counted for each) up to
// which the sequences read the prefix one by one.
constexpr long long kWalkTokens = 4096;
constexpr double kDenseCost = 1.5;  // an FP32 tile in packed ones

constexpr int kTile = 32;           // tokens of a tile: FP32 rows or packed slots
constexpr float kLimit = 65000.0f;  // scaled keys and values stay below this
constexpr float kLow = 0.125f;      // a first tile of smaller keys or values is scaled up
constexpr float kSlack = 2.0f;      // of the lazy rescale, log2 units
constexpr float kUp = 12.0f;        // P's largest value when the reference moves, log2 units

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

template <int DC, int RT, int WM, int WT>
struct Config {
    static constexpr int WAVES = WM * WT;
    static constexpr bool ALONE = WM == 1;  // every wave stages for itself
    // two tiles in turn, so that staging one needs no wait for the readers of the other, where two waves per SIMD fit
    static constexpr int NBUF = !ALONE && WT == 1 && 2 * TileLds<DC>::BYTES * 8 / WM <= kLds - 256 ? 2 : 1;
    static constexpr int TILES = NBUF * WT;
    static constexpr int PEAKS = ALONE ? 2 * WT : 2 * NBUF;
    static constexpr int LDS = TILES * TileLds<DC>::BYTES + 16 * ((PEAKS + 3) / 4);
    static constexpr int PER_CU = kLds / LDS < 8 / WAVES ? kLds / LDS : 8 / WAVES;
    static constexpr int PER_EU = PER_CU * WAVES >= 8 ? 2 : 1;
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

// (hi, lo) of two values, both truncated: hi + lo is x to 21 bits.
__device__ __forceinline__ uint2 parts(const float x0, const float x1) {
    const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    const float r0 = fma_mix_lo(hi, -1.0f, x0), r1 = fma_mix_hi(hi, -1.0f, x1);
    return make_uint2(hi, __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1)));
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

typedef uint32_t un_u4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t un_u2 __attribute__((ext_vector_type(2), aligned(2)));

// One workgroup's share [t0, t1) of the prefix's tiles of one kind, for rows row0 .. of one KV head. DC: 32-channel
// chunks of a head. RT: 16-row tiles per wave. WM x WT waves: WM share a tile and take other rows, WT take other tiles.
template <int DC, int RT, int WM, int WT, bool PACKED>
__device__ __forceinline__ void shared_body(const SharedArgs& a, char* lds, const Tiers& t, const int kvh,
                                            const int row0, const int rows, const int t0, const int t1,
                                            const int slot) {
    using C = Config<DC, RT, WM, WT>;
    using L = TileLds<DC>;
    constexpr int NK = (DC + WM - 1) / WM, NV = NK;  // K (V) units of a wave: 64 lanes x (4 tokens x 4 channels)
    constexpr bool APART = WM >= 2 * DC;             // enough waves for K and V apart
    const int lane = threadIdx.x & 63;
    const int wave = scalar(static_cast<int>(threadIdx.x) >> 6);
    const int wm = wave % WM, wt = wave / WM;
    const int n = lane & 15, g = lane >> 4;
    const int G = a.Hq / a.Hkv;
    const int D = a.D;
    const size_t Hkv = static_cast<size_t>(a.Hkv);
    // Waves that share a tile take its units in turn (DC: none): K's from the first wave on, V's from the wave behind
    // them, or from the last wave backwards.
    auto kunit = [&](const int i) { return wm + WM * i; };
    auto vunit = [&](const int i) { return APART ? (wm >= DC ? wm - DC : DC) : WM - 1 - wm + WM * i; };

    // K units: lane = (token quad, channel quad); V units the other way round,
    // so that the writes of V's transposed rows spread over the banks.
    const int ktq = lane >> 3, kcq = lane & 7;
    const int vtq = lane & 7, vcq = lane >> 3;
    const bool f16m = a.meta_fp16 != 0;

    // The tile in flight, as it lies in memory.
    mf_u4 kx[NK][PACKED ? 3 : 4];  // packed: words, scale, zero; FP32: 4 tokens
    mf_u4 vx[NV][PACKED ? 1 : 4];
    uint2 idv = make_uint2(0u, 0u);
    uint32_t vm = 0u;              // packed: V scale (lanes 0-31) or zero (lanes 32-63) of token lane % 32
    auto fetch = [&](const int tile) {
        const int s0 = kTile * tile;
        if constexpr (PACKED) {
            const int last = t.slots - 1;
            const int sl = min(s0 + (lane & 31), last);
            idv = *reinterpret_cast<const uint2*>(t.ids + sl);
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int u = kunit(i);
                if (u >= DC) break;
                const int c = min(32 * u + 4 * kcq, D - 4);
                const int s = min(s0 + 4 * ktq, last);
                const size_t km = static_cast<size_t>(a.kgs == 32 ? s >> 5 : s >> 4) * Hkv * D + c;
                kx[i][0] = *reinterpret_cast<const un_u4*>(t.kp + static_cast<size_t>(s >> 4) * Hkv * D + c);
                if (!f16m) {
                    kx[i][1] = *reinterpret_cast<const un_u4*>(t.ks + 4 * km);
                    kx[i][2] = *reinterpret_cast<const un_u4*>(t.kz + 4 * km);
                } else {
                    const un_u2 ps = *reinterpret_cast<const un_u2*>(t.ks + 2 * km);
                    const un_u2 pz = *reinterpret_cast<const un_u2*>(t.kz + 2 * km);
                    kx[i][1] = mf_u4{ps[0], ps[1], 0u, 0u};
                    kx[i][2] = mf_u4{pz[0], pz[1], 0u, 0u};
                }
            }
            const char* vmp = lane < 32 ? t.vs : t.vz;
            if (vunit(0) != 0)
                ;  // another wave's
            else if (!f16m)
                vm = *reinterpret_cast<const uint32_t*>(vmp + 4 * (sl * Hkv));
            else
                vm = *reinterpret_cast<const uint16_t*>(vmp + 2 * (sl * Hkv));
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int u = vunit(i);
                if (u >= DC) break;
                const int c = min(32 * u + 4 * vcq, D - 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    vx[i][0][j] = t.vp[static_cast<size_t>(min(s0 + 4 * vtq + j, last)) * Hkv * (D / 16) + (c >> 4)];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int u = kunit(i);
                if (u >= DC) break;
                const int c = min(32 * u + 4 * kcq, D - 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    kx[i][j] = *reinterpret_cast<const un_u4*>(t.dk + min(s0 + 4 * ktq + j, t.nd - 1) * Hkv * D + c);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int u = vunit(i);
                if (u >= DC) break;
                const int c = min(32 * u + 4 * vcq, D - 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    vx[i][j] = *reinterpret_cast<const un_u4*>(t.dv + min(s0 + 4 * vtq + j, t.nd - 1) * Hkv * D + c);
            }
        }
    };
    // Bit j: token j of the fetched tile is attended.
    auto mask_of = [&](const int tile) -> uint32_t {
        const int left = (PACKED ? t.slots : t.nd) - kTile * tile;
        const uint32_t in = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
        if constexpr (PACKED) return static_cast<uint32_t>(__ballot((idv.x & idv.y) != 0xffffffffu)) & in;
        return in;
    };

    float* peak = reinterpret_cast<float*>(lds + C::TILES * L::BYTES);  // [buffer or wave][key, value]
    // A tile's largest key or value where it asks for another scale: too large for f16 at this one, or (first) any.
    // The peaks only grow and so do the exponents after the first: none is ever cleared. Positive floats order like their bits. (An infinity has no scale that helps: it is left to make
    // NaN of what reads it.)
    auto report = [&](const float x, const float back, const bool first, float* to) {
        if (__ballot(x >= kLimit || (first && x > 0.0f)))
            if ((x >= kLimit || (first && x > 0.0f)) && x < __builtin_huge_valf())
                atomicMax(reinterpret_cast<int*>(to), __float_as_int(fminf(x * back, 3.0e38f)));
    };

    // f16 parts of the fetched K (scaled by 2^(4 - ke)).
    auto stage_k = [&](char* tl, const uint32_t mask, const int ke, const bool first, float* to) {
        const float ksc = __builtin_amdgcn_ldexpf(16.0f, -ke);
        const uint32_t mine = (mask >> (4 * ktq)) & 15u;
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int u = kunit(i);
            if (u >= DC) break;
            const int c0 = 32 * u + 4 * kcq;
            float x[4][4];  // [token][channel]
            if constexpr (PACKED) {
                // no attended token: the block's scale and zero may be anything
                const bool any = mine != 0u && c0 < D;
                float sc[4], zr[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t ws = kx[i][1][e], wz = kx[i][2][e];
                    const uint32_t hs = kx[i][1][e >> 1], hz = kx[i][2][e >> 1];
                    const float s = f16m ? ((e & 1) ? half_hi(hs) : half_lo(hs)) : __uint_as_float(ws);
                    const float z = f16m ? ((e & 1) ? half_hi(hz) : half_lo(hz)) : __uint_as_float(wz);
                    sc[e] = any ? s * ksc : 0.0f;
                    zr[e] = any ? z * ksc : 0.0f;
                    mx = fmax_abs_nn(mx, fmax_abs_nn(zr[e], __builtin_fmaf(3.0f, sc[e], zr[e])));
                }
                // the quad's codes, one byte per channel, then one code per byte
                const uint32_t b = 0x0c0c0400u + 0x0101u * (ktq & 3);
                const uint32_t lo = __builtin_amdgcn_perm(kx[i][0][1], kx[i][0][0], b);
                const uint32_t hi = __builtin_amdgcn_perm(kx[i][0][3], kx[i][0][2], b);
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
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[j][e] = ((mine >> j) & 1u) && c0 < D ? __uint_as_float(kx[i][j][e]) * ksc : 0.0f;
                        mx = fmaxf(mx, fabsf(x[j][e]));
                    }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint2 p = parts(x[j][0], x[j][1]), q = parts(x[j][2], x[j][3]);
                char* d = tl + (4 * ktq + j) * L::KS + 2 * c0;
                *reinterpret_cast<uint2*>(d + L::KHI) = make_uint2(p.x, q.x);
                *reinterpret_cast<uint2*>(d + L::KLO) = make_uint2(p.y, q.y);
            }
        }
        report(mx, __builtin_amdgcn_ldexpf(0.0625f, ke), first, to);
    };
    // Packed: the centred codes (2 q - 3) 4^(c % 4), exact, of channels c; FP32: f16 parts of V 2^(4 - ve). Token quad
    // vtq sits in the MFMA order: 8 tokens per lane group, its half by the 16-token tile.
    auto stage_v = [&](char* tl, const uint32_t mask, const int ve, const bool first, float* to) {
        const float vsc = __builtin_amdgcn_ldexpf(16.0f, -ve);
        const uint32_t mine = (mask >> (4 * vtq)) & 15u;
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = vunit(i);
            if (u >= DC) break;
            const int c0 = 32 * u + 4 * vcq;
            char* d = tl + c0 * L::VS + 16 * (vtq & 3) + 8 * (vtq >> 2);
            if constexpr (PACKED) {
                // channels past head_dim hold codes of others, in columns that are not stored
                const uint32_t b = 0x0c040c00u + 0x00010001u * (vcq & 3);
                const uint32_t y0 = __builtin_amdgcn_perm(vx[i][0][1], vx[i][0][0], b) << 1;
                const uint32_t y1 = __builtin_amdgcn_perm(vx[i][0][3], vx[i][0][2], b) << 1;
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
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        y[j] = ((mine >> j) & 1u) && c0 < D ? __uint_as_float(vx[i][j][e]) * vsc : 0.0f;
                        mx = fmaxf(mx, fabsf(y[j]));
                    }
                    const uint2 p = parts(y[0], y[1]), q = parts(y[2], y[3]);
                    *reinterpret_cast<uint2*>(d + e * L::VS + L::V) = make_uint2(p.x, q.x);
                    *reinterpret_cast<uint2*>(d + e * L::VS + L::VLO) = make_uint2(p.y, q.y);
                }
            }
        }
        if constexpr (!PACKED) report(mx, __builtin_amdgcn_ldexpf(0.0625f, ve), first, to);
    };
    // Packed: V's scale 2^-ve and the zero of the centred codes, vz + 1.5 vs, of the tile's tokens (zeros where masked).
    auto stage_vmeta = [&](char* tl, const uint32_t mask, const int ve, const bool first, float* to) {
        const float x = f16m ? half_lo(vm) : __uint_as_float(vm);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        float y = lane < 32 ? x : __builtin_fmaf(1.5f, __uint_as_float(sw[0]), x);
        y = ((mask >> (lane & 31)) & 1u) ? __builtin_amdgcn_ldexpf(y, -ve) : 0.0f;
        reinterpret_cast<float*>(tl + L::VMETA)[lane] = y;
        // a scale up to 2 2^ve stays in reach (P <= 2^14); reported in units of kLimit / 2
        report(lane < 32 ? fabsf(y) * (0.5f * kLimit) : 0.0f, __builtin_amdgcn_ldexpf(2.0f / kLimit, ve), first, to);
    };

    // The first tile's loads go out before the queries'.
    if (t0 + wt < t1) fetch(t0 + wt);

    // Q' = Q 2^(12 - e), e the exponent of the row's largest value, as the QK B operand: row n of row tile rt, channels
    // 32 s + 8 g .. + 7.
    mf_u4 qh[RT][DC], ql[RT][DC];
    float crow[RT];  // log2 units per unit of the product
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = row0 + 16 * (RT * wm + rt) + n;
        const bool live = r < rows;
        const int seq = live ? r / G : 0;
        const int h = kvh * G + (live ? r % G : 0);
        const float* q = global_ptr(a.seqs[seq].Q) + static_cast<size_t>(h) * D;
        float x[DC][8];
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < DC; ++s) {
            const int c = 32 * s + 8 * g;
            const bool in = live && c < D;
            const un_u4 y = *reinterpret_cast<const un_u4*>(q + min(c, D - 8));
            const un_u4 z = *reinterpret_cast<const un_u4*>(q + min(c, D - 8) + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[s][j] = in ? __uint_as_float(y[j]) : 0.0f;
                x[s][4 + j] = in ? __uint_as_float(z[j]) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(x[s][j]));
        }
        mx = xrow_max(mx);
        const int e = (mx > 0.0f) ? __builtin_amdgcn_frexp_expf(mx) : 0;
#pragma unroll
        for (int s = 0; s < DC; ++s) {
            uint2 p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                p[j] = parts(__builtin_amdgcn_ldexpf(x[s][2 * j], 12 - e), __builtin_amdgcn_ldexpf(x[s][2 * j + 1], 12 - e));
            qh[rt][s] = mf_u4{p[0].x, p[1].x, p[2].x, p[3].x};
            ql[rt][s] = mf_u4{p[0].y, p[1].y, p[2].y, p[3].y};
        }
        crow[rt] = __builtin_amdgcn_ldexpf(a.scale2, e - 16);
    }

    mf_f4 acc[RT][2 * DC];
    float mr[RT], l[RT], pz[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        mr[rt] = -3.0e38f;
        l[rt] = 0.0f;
        pz[rt] = 0.0f;
#pragma unroll
        for (int s = 0; s < 2 * DC; ++s) acc[rt][s] = mf_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // Exponents of the scales of K and V, and whether no tile has set them yet: of the workgroup, or of each wave
    // that stages for itself.
    int k_exp = 0, v_exp = 0;
    bool kfirst = true, vfirst = true;
    float* peaks = peak + (C::ALONE ? 2 * wave : 0);
    if (threadIdx.x < C::PEAKS) peak[threadIdx.x] = 0.0f;
    lds_barrier();
    auto sync = [&]() {
        if constexpr (C::ALONE)
            wave_lds_sync();
        else
            lds_barrier();
    };

    // The new exponents that the tile's peaks ask for; true if they changed.
    auto adjust = [&](const float* pk) -> bool {
        const float pk_k = pk[0], pk_v = pk[1];
        int kn = k_exp, vn = v_exp;
        if (__ballot(pk_k > 0.0f)) {
            const int e = scalar(__builtin_amdgcn_frexp_expf(pk_k)) - 11;  // largest scaled key below 2^15
            if (e > k_exp || (kfirst && __ballot(pk_k < kLow))) kn = e;
            kfirst = false;
        }
        if (__ballot(pk_v > 0.0f)) {
            const int e = scalar(__builtin_amdgcn_frexp_expf(pk_v)) - (PACKED ? 0 : 11);
            if (e > v_exp + (PACKED ? 1 : 0) || (vfirst && __ballot(pk_v < kLow))) vn = e;
            vfirst = false;
        }
        if (kn == k_exp && vn == v_exp) return false;
        const float f = __builtin_amdgcn_ldexpf(1.0f, v_exp - vn);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            pz[rt] *= f;
#pragma unroll
            for (int s = 0; s < 2 * DC; ++s) acc[rt][s] *= f;
        }
        k_exp = kn;
        v_exp = vn;
        return true;
    };

    // QK of the staged tile.
    auto qk = [&](const char* tl, mf_f4 (&d)[RT][2]) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 2; ++i) d[rt][i] = mf_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < DC; ++s) {
            mf_u4 kh[2], kl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const char* p = tl + (16 * i + n) * L::KS + 64 * s + 16 * g;
                kh[i] = *reinterpret_cast<const mf_u4*>(p + L::KHI);
                kl[i] = *reinterpret_cast<const mf_u4*>(p + L::KLO);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) d[rt][i] = mfma16x16x32(kh[i], ql[rt][s], d[rt][i]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) d[rt][i] = mfma16x16x32(kl[i], qh[rt][s], d[rt][i]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) d[rt][i] = mfma16x16x32(kh[i], qh[rt][s], d[rt][i]);
        }
    };
    // Softmax of the tile's logits, P (packed: P times V's scale) as the PV A operand.
    auto softmax = [&](const char* tl, const uint32_t mask, mf_f4 (&d)[RT][2], mf_u4 (&ph)[RT], mf_u4 (&pl)[RT]) {
        mf_f4 vs[2], vz[2];
        if constexpr (PACKED) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                vs[i] = *reinterpret_cast<const mf_f4*>(tl + L::VMETA + 64 * i + 16 * g);
                vz[i] = *reinterpret_cast<const mf_f4*>(tl + L::VMETA + 128 + 64 * i + 16 * g);
            }
        }
        if (mask != 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = (mask >> (16 * i + 4 * g + r)) & 1u;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) d[rt][i][r] = in ? d[rt][i][r] : kNegInf;
                }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float c = __builtin_amdgcn_ldexpf(crow[rt], k_exp);
            float mx = fmaxf(fmaxf(fmaxf(d[rt][0][0], d[rt][0][1]), fmaxf(d[rt][0][2], d[rt][0][3])),
                             fmaxf(fmaxf(d[rt][1][0], d[rt][1][1]), fmaxf(d[rt][1][2], d[rt][1][3])));
            mx = __builtin_fmaf(mx, c, -kUp);
            // the reference moves only when a row's maximum passes it by more than the slack
            if (__ballot(mx > mr[rt] + kSlack)) {
                mx = xrow_max(mx);
                const bool up = mx > mr[rt] + kSlack;
                const float mn = up ? mx : mr[rt];
                const float al = up ? __builtin_amdgcn_exp2f(mr[rt] - mn) : 1.0f;
                l[rt] *= al;
                pz[rt] *= al;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float ar = __shfl(al, 4 * g + r, 64);
#pragma unroll
                    for (int q = 0; q < 2 * DC; ++q) acc[rt][q][r] *= ar;
                }
                mr[rt] = mn;
            }
            float p[2][4];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(d[rt][i][r], c, -mr[rt]));
                    sum += p[i][r];
                    if constexpr (PACKED) {
                        pz[rt] = __builtin_fmaf(p[i][r], vz[i][r], pz[rt]);
                        p[i][r] *= vs[i][r];
                    }
                }
            l[rt] += sum;
            const uint2 p0 = parts(p[0][0], p[0][1]), p1 = parts(p[0][2], p[0][3]);
            const uint2 p2 = parts(p[1][0], p[1][1]), p3 = parts(p[1][2], p[1][3]);
            ph[rt] = mf_u4{p0.x, p1.x, p2.x, p3.x};
            pl[rt] = mf_u4{p0.y, p1.y, p2.y, p3.y};
        }
    };
    auto pv = [&](const char* tl, const mf_u4 (&ph)[RT], const mf_u4 (&pl)[RT]) {
#pragma unroll
        for (int q = 0; q < 2 * DC; ++q) {
            const char* p = tl + (16 * q + n) * L::VS + 16 * g;
            const mf_u4 vh = *reinterpret_cast<const mf_u4*>(p + L::V);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][q] = mfma16x16x32(pl[rt], vh, acc[rt][q]);
            if constexpr (!PACKED) {
                const mf_u4 vl = *reinterpret_cast<const mf_u4*>(p + L::VLO);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][q] = mfma16x16x32(ph[rt], vl, acc[rt][q]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][q] = mfma16x16x32(ph[rt], vh, acc[rt][q]);
        }
    };


    auto stage = [&](char* tl, const uint32_t mask, float* pk) {
        stage_k(tl, mask, k_exp, kfirst, pk);
        stage_v(tl, mask, v_exp, vfirst, pk + 1);
        if constexpr (PACKED)
            if (vunit(0) == 0) stage_vmeta(tl, mask, v_exp, vfirst, pk + 1);
    };
    int buf = 0;
    for (int tb = t0; tb < t1; tb += WT) {
        const int tile = tb + wt;
        const bool mine = tile < t1;
        char* tl = lds + (C::NBUF * wt + buf) * L::BYTES;
        float* pk = peaks + 2 * buf;
        if constexpr (C::NBUF == 1) sync();  // the last tile's readers are done
        const uint32_t mask = mine ? mask_of(tile) : 0u;
        if (mine) stage(tl, mask, pk);
        if (tile + WT < t1) fetch(tile + WT);
        sync();
        if (adjust(pk)) {
            // keys or values outside what f16 holds well at this scale: the tile again
            sync();
            if (mine) {
                fetch(tile);
                stage(tl, mask, pk);
            }
            if (tile + WT < t1) fetch(tile + WT);
            sync();
        }
        if constexpr (C::NBUF == 2) buf ^= 1;
        if (!mine) continue;
        mf_f4 d[RT][2];
        mf_u4 ph[RT], pl[RT];
        qk(tl, d);
        softmax(tl, mask, d, ph, pl);
        pv(tl, ph, pl);
    }

    // The partial in units of V: acc holds 16 V 2^-v_exp (FP32 tiles), or 2 4^(c % 4) of it without the centred zero.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = xrow_sum(l[rt]);
    const float back = __builtin_amdgcn_ldexpf(1.0f, v_exp - (PACKED ? 1 + 2 * (n & 3) : 4));
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float z = PACKED ? __builtin_amdgcn_ldexpf(xrow_sum(pz[rt]), v_exp) : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float zr = PACKED ? __shfl(z, 4 * g + r, 64) : 0.0f;
#pragma unroll
            for (int q = 0; q < 2 * DC; ++q) acc[rt][q][r] = __builtin_fmaf(acc[rt][q][r], back, zr);
        }
    }
    auto partial = [&](const int r) {  // index of row r's partial
        const int seq = r / G;
        const int h = kvh * G + r % G;
        const int ns = a.slot_base[seq + 1] - a.slot_base[seq];
        return static_cast<size_t>(a.slot_base[seq]) * a.Hq + static_cast<size_t>(h) * ns + (ns - a.prefix_slots + slot);
    };
    if constexpr (WT == 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int rn = row0 + 16 * (RT * wm + rt) + n;
            if (g == 0 && rn < rows) {
                const size_t pi = partial(rn);
                a.ml[2 * pi] = l[rt] > 0.0f ? mr[rt] : kNegInf;
                a.ml[2 * pi + 1] = l[rt];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int rr = row0 + 16 * (RT * wm + rt) + 4 * g + r;
                if (rr >= rows) continue;
                float* o = a.acc + partial(rr) * D;
#pragma unroll
                for (int q = 0; q < 2 * DC; ++q)
                    if (16 * q < D) o[16 * q + n] = acc[rt][q][r];
            }
        }
    } else {
        // The waves of one row tile took other tokens: joined in LDS.
        constexpr int RW = 16 * RT;                 // rows of a wave
        constexpr int LINE = 32 * DC + 4;           // floats per row: accumulators, reference, sum
        static_assert(WM * WT * RW * LINE * 4 <= C::TILES * L::BYTES, "the merge fits in the tiles' LDS");
        lds_barrier();
        float* my = reinterpret_cast<float*>(lds) + wave * RW * LINE;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (g == 0) {
                my[(16 * rt + n) * LINE + 32 * DC] = mr[rt];
                my[(16 * rt + n) * LINE + 32 * DC + 1] = l[rt];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int q = 0; q < 2 * DC; ++q) my[(16 * rt + 4 * g + r) * LINE + 16 * q + n] = acc[rt][q][r];
        }
        lds_barrier();
        for (int idx = threadIdx.x; idx < WM * RW * 32 * DC; idx += 64 * WM * WT) {
            const int row = idx / (32 * DC), c = idx - row * 32 * DC;  // row of the workgroup, channel
            const int rr = row0 + row;
            if (rr >= rows || c >= D) continue;
            const float* x = reinterpret_cast<const float*>(lds) + row * LINE;
            constexpr int STEP = WM * RW * LINE;  // to the next wave of the same rows
            float M = -3.0e38f;
#pragma unroll
            for (int w = 0; w < WT; ++w) M = fmaxf(M, x[w * STEP + 32 * DC]);
            float A = 0.0f, Ls = 0.0f;
#pragma unroll
            for (int w = 0; w < WT; ++w) {
                const float f = __builtin_amdgcn_exp2f(x[w * STEP + 32 * DC] - M);
                A = __builtin_fmaf(f, x[w * STEP + c], A);
                Ls = __builtin_fmaf(f, x[w * STEP + 32 * DC + 1], Ls);
            }
            const size_t pi = partial(rr);
            a.acc[pi * D + c] = A;
            if (c == 0) {
                a.ml[2 * pi] = Ls > 0.0f ? M : kNegInf;
                a.ml[2 * pi + 1] = Ls;
            }
        }
    }
}

// First of `count` items of part i of `parts`.
__device__ __forceinline__ int share(const int count, const int i, const int parts) {
    return scalar(static_cast<int>(static_cast<long long>(count) * i / parts));
}

// Grid: slots x (KV heads x row chunks); slot s of all heads and chunks on XCD
// s % 8, back to back, so that a tile's lines come from memory once. Slots
// [0, packed_slots) share the packed tiles, the others the FP32 ones.
template <int DC, int RT, int WM, int WT>
__global__ void __launch_bounds__(64 * WM * WT) __attribute__((amdgpu_waves_per_eu(Config<DC, RT, WM, WT>::PER_EU)))
attn_shared_kernel(const SharedArgs a) {
    __shared__ __align__(16) char lds[Config<DC, RT, WM, WT>::LDS];
    const unsigned id = blockIdx.x;
    const unsigned q = id >> 3;
    const unsigned hc = static_cast<unsigned>(a.Hkv * a.chunks);
    const int hz = static_cast<int>(q % hc);
    const int s = static_cast<int>((q / hc) * 8 + (id & 7));
    if (s >= a.prefix_slots) return;
    const int kvh = hz / a.chunks, chunk = hz - kvh * a.chunks;
    const int rows = a.nseq * (a.Hq / a.Hkv), row0 = chunk * 16 * RT * WM;
    const Tiers t = tiers_of(a, kvh);
    if (s < a.packed_slots) {
        const int tiles = (t.slots + kTile - 1) / kTile;
        shared_body<DC, RT, WM, WT, true>(a, lds, t, kvh, row0, rows, share(tiles, s, a.packed_slots),
                                          share(tiles, s + 1, a.packed_slots), s);
    } else {
        const int tiles = (t.nd + kTile - 1) / kTile, nd = a.prefix_slots - a.packed_slots;
        shared_body<DC, RT, WM, WT, false>(a, lds, t, kvh, row0, rows, share(tiles, s - a.packed_slots, nd),
                                           share(tiles, s - a.packed_slots + 1, nd), s);
    }
}

template <int DC, int RT, int WM, int WT>
int launch(SharedArgs a, const int rows, hipStream_t st) {
    a.chunks = (rows + 16 * RT * WM - 1) / (16 * RT * WM);
    const long long wgs = static_cast<long long>((a.prefix_slots + 7) / 8) * 8 * a.Hkv * a.chunks;
    if (wgs > 0x00ffffffLL) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "attention grid too large");
    hipLaunchKernelGGL((attn_shared_kernel<DC, RT, WM, WT>), dim3(static_cast<unsigned>(wgs)), dim3(64 * WM * WT), 0, st, a);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

// What a workgroup takes, by rows per KV head and 32-channel chunks of a head:
// its rows, its tiles at once, and how many workgroups a CU holds.
struct Shape {
    int rows, tiles, per_cu;
};
enum Size { kOne, kTwo, kFour, kEight };  // row tiles of 32 (kOne: 16), shared by as many waves

Size size_for(const int rows) { return rows <= 16 ? kOne : rows <= 64 ? kTwo : rows <= 128 ? kFour : kEight; }

template <int DC, int RT, int WM, int WT, typename F>
auto with(F&& f) {
    return f(std::integral_constant<int, DC>{}, std::integral_constant<int, RT>{}, std::integral_constant<int, WM>{},
             std::integral_constant<int, WT>{});
}
template <int DC, typename F>
auto for_rows(const int rows, F&& f) {
    constexpr int RT = DC <= 4 ? 2 : 1;
    switch (size_for(rows)) {
    case kOne: return with<DC, 1, 1, (DC <= 4 ? 4 : 2)>(f);
    case kTwo: return with<DC, RT, 2, 2>(f);
    case kFour: return with<DC, RT, 4, 1>(f);
    default: return with<DC, RT, 8, 1>(f);
    }
}
template <typename F>
auto for_shape(const int D, const int rows, F&& f) {
    if (D <= 64) return for_rows<2>(rows, f);
    if (D <= 96) return for_rows<3>(rows, f);
    if (D <= 128) return for_rows<4>(rows, f);
    if (D <= 192) return for_rows<6>(rows, f);
    return for_rows<8>(rows, f);
}

Shape shape_of(const int D, const int rows) {
    return for_shape(D, rows, [](auto dc, auto rt, auto wm, auto wt) {
        using C = Config<dc.value, rt.value, wm.value, wt.value>;
        return Shape{16 * rt.value * wm.value, wt.value, C::PER_CU};
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
    p.per_seq = tokens > 0 && nseq <= kMaxBatchSeqs / 2 && nseq * tokens <= kWalkTokens ? 2 : 1;
    tt_decode_seq entries[kMaxBatchSeqs];
    for (int i = 0; i < nseq; ++i) {
        entries[p.per_seq * i] = seqs[i];
        if (p.per_seq == 2) {
            entries[2 * i + 1] = prefix;
            entries[2 * i + 1].mean_attn_weights = nullptr;
        }
    }
    p.entries = own_plan(entries, p.per_seq * nseq, Hq, Hkv, D, kgs, meta_fp16);
    if (p.per_seq == 1 && tokens > 0) {
        const Shape sh = shape_of(D, rows);
        const long long groups = static_cast<long long>(Hkv) * ((rows + sh.rows - 1) / sh.rows);
        // one round of workgroups, each kind's share by what its tiles cost
        const long long slots = std::max<long long>(1, 256LL * sh.per_cu / groups);
        const double cost = packed + kDenseCost * dense;
        long long np = packed ? std::max<long long>(1, std::llround(slots * packed / cost)) : 0;
        np = std::min(np, (packed + sh.tiles - 1) / sh.tiles);
        long long nd = dense ? std::max<long long>(1, slots - np) : 0;
        nd = std::min(nd, (dense + sh.tiles - 1) / sh.tiles);
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
        const int rc = for_shape(D, rows, [&](auto dc, auto rt, auto wm, auto wt) {
            return launch<dc.value, rt.value, wm.value, wt.value>(a, rows, stream);
        });
        if (rc) return rc;
    }
    const int rc = own_launch(plan, prefix, seqs_dev, Hq, Hkv, D, kgs, meta_fp16, ws, stream);
    if (rc) return rc;
    return batch_finalize(b, seqs_dev, Hq, D, kgs, ws, stream, true);
}

}  // namespace tt
