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

namespace tt {
namespace {

constexpr int kTile = 32;           // tokens of a tile: FP32 rows or packed slots
constexpr float kLimit = 65000.0f;  // largest scaled key or value whose f16 parts are finite
constexpr float kLow = 0.125f;      // a first tile of smaller keys or values is scaled up
constexpr float kSlack = 2.0f;      // of the lazy rescale, log2 units
constexpr float kUp = 12.0f;        // P's largest value when the reference moves, log2 units

// LDS of one tile: K as [token][channel], V as [channel][token in MFMA order],
// high and low parts, and each token's bias (0, or -inf where masked). The row
// strides put the 16-byte reads of eight lanes and the 8-byte writes of
// sixteen in distinct banks.
template <int DC>
struct TileLds {
    static constexpr int KS = 64 * DC + 16;           // bytes per K row
    static constexpr int VS = 80;                     // bytes per V row
    static constexpr int KHI = 0;
    static constexpr int KLO = KHI + kTile * KS;
    static constexpr int VHI = KLO + kTile * KS;
    static constexpr int VLO = VHI + 32 * DC * VS;
    static constexpr int BIAS = VLO + 32 * DC * VS;   // [32] f32 in token order
    static constexpr int BYTES = BIAS + kTile * 4;
};

struct SharedArgs {
    const tt_decode_seq* __restrict__ seqs;
    tt_decode_seq prefix;
    float* ml;
    float* acc;
    float* logits;
    float scale2;         // log2(e) / sqrt(head_dim)
    int nseq, Hq, Hkv, D, kgs, meta_fp16;
    int prefix_slots;
    int chunks;           // row chunks per KV head
    int total;            // slots of the launch: prefix_slots, or the own slots of all sequences
    int slot_base[kMaxBatchSeqs + 1];
    int own_base[kMaxBatchSeqs + 1];
    int tok_base[kMaxBatchSeqs + 1];
};

__device__ __forceinline__ int find_seq(const int* base, const int n, const int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// (hi, lo) of two values, both truncated: hi + lo is x to 21 bits.
__device__ __forceinline__ uint2 parts(const float x0, const float x1) {
    const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    const float r0 = fma_mix_lo(hi, -1.0f, x0), r1 = fma_mix_hi(hi, -1.0f, x1);
    return make_uint2(hi, __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1)));
}

__device__ __forceinline__ float half_lo(const uint32_t x) { return f16_to_f32(static_cast<uint16_t>(x & 0xffffu)); }
__device__ __forceinline__ float half_hi(const uint32_t x) { return f16_to_f32(static_cast<uint16_t>(x >> 16)); }

// The tiers of one work item, for one KV head.
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
    int td, tiles;    // FP32 tiles, all tiles
};

__device__ __forceinline__ Tiers tiers_of(const tt_decode_seq& d, const SharedArgs& a, const int kvh) {
    const int m = a.meta_fp16 ? 2 : 4;
    Tiers t;
    t.dk = global_ptr(d.dense_K) + static_cast<size_t>(kvh) * a.D;
    t.dv = global_ptr(d.dense_V) + static_cast<size_t>(kvh) * a.D;
    t.kp = reinterpret_cast<const uint32_t*>(global_ptr(d.PBS_K_Packed)) + static_cast<size_t>(kvh) * a.D;
    t.ks = static_cast<const char*>(global_ptr<const char>(reinterpret_cast<uint64_t>(d.PBS_K_Scales))) + static_cast<size_t>(kvh) * a.D * m;
    t.kz = static_cast<const char*>(global_ptr<const char>(reinterpret_cast<uint64_t>(d.PBS_K_Zeroes))) + static_cast<size_t>(kvh) * a.D * m;
    t.vp = reinterpret_cast<const uint32_t*>(global_ptr(d.PBS_V_Packed)) + static_cast<size_t>(kvh) * (a.D / 16);
    t.vs = static_cast<const char*>(global_ptr<const char>(reinterpret_cast<uint64_t>(d.PBS_V_Scales))) + static_cast<size_t>(kvh) * m;
    t.vz = static_cast<const char*>(global_ptr<const char>(reinterpret_cast<uint64_t>(d.PBS_V_Zeroes))) + static_cast<size_t>(kvh) * m;
    t.ids = global_ptr(d.PBS_token_ids);
    t.nd = scalar(d.dense_count);
    t.slots = scalar(d.num_blocks) * a.kgs;
    t.td = (t.nd + kTile - 1) / kTile;
    t.tiles = t.td + (t.slots + kTile - 1) / kTile;
    return t;
}

// A tile's data on its way from memory: the units of one wave. A unit is 64
// lanes x (4 tokens x 4 channels) of K or of V: 32 tokens, 32 channels.
// Everything stays in its stored form until the tile is staged.
template <int NU>
struct Raw {
    mf_u4 x[NU][4];    // FP32 tile: 4 tokens; packed K: [0] words, [1] scale, [2] zero; packed V: [0] words
    mf_u4 vm[2];       // packed V: scale and zero of the lane's tokens
    uint2 ids[2][4];   // packed: ids of the lane's tokens (K units, V units)
};

// DC: 32-channel chunks of a head (head_dim padded). RT: 16-row tiles per wave. WM x WT waves: WM share a tile's
// tokens and take other rows, WT take other tiles.
template <int DC, int RT, int WM, int WT>
__device__ __forceinline__ void shared_body(const SharedArgs& a, char* lds, const Tiers& t, const int kvh,
                                            const int row0, const int rows, const int only, const int t0, const int t1,
                                            const int slot) {
    using L = TileLds<DC>;
    constexpr int NU = (2 * DC + WM - 1) / WM;     // units per wave
    const int lane = threadIdx.x & 63;
    const int wave = scalar(static_cast<int>(threadIdx.x) >> 6);
    const int wm = wave % WM, wt = wave / WM;
    const int n = lane & 15, g = lane >> 4;
    const int G = a.Hq / a.Hkv;
    const int D = a.D;
    char* tl = lds + wt * L::BYTES;
    // largest key and value past the limit, and of the tiles up to the first with any that is not zero
    float* over = reinterpret_cast<float*>(lds + WT * L::BYTES);
    float* low = over + 2;

    // K units: lane = (token quad, channel quad); V units the other way round,
    // so that the writes of V's transposed rows spread over the banks.
    const int ktq = lane >> 3, kcq = lane & 7;
    const int vtq = lane & 7, vcq = lane >> 3;
    const int m = a.meta_fp16 ? 2 : 4;

    Raw<NU> raw;
    auto fetch = [&](const int tile) {
        if (tile < t.td) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int u = wm + WM * i;
                if (u >= 2 * DC) break;
                const bool isk = u < DC;
                const int c = 32 * (isk ? u : u - DC) + 4 * (isk ? kcq : vcq);
                const int tok = kTile * tile + 4 * (isk ? ktq : vtq);
                const float* base = isk ? t.dk : t.dv;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    raw.x[i][j] = mf_u4{0u, 0u, 0u, 0u};
                    if (tok + j < t.nd && c < D) {
                        typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
                        raw.x[i][j] = *reinterpret_cast<const u4*>(base + static_cast<size_t>(tok + j) * a.Hkv * D + c);
                    }
                }
            }
            return;
        }
        const int s0 = kTile * (tile - t.td);  // first slot
        const int last = t.slots - 1;
        typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
        typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = wm + WM * i;
            if (u >= 2 * DC) break;
            if (u < DC) {
                const int c = min(32 * u + 4 * kcq, D - 4);
                const int s = min(s0 + 4 * ktq, last);
                const size_t kw = static_cast<size_t>(s >> 4) * a.Hkv * D + c;
                const size_t km = static_cast<size_t>(s / a.kgs) * a.Hkv * D + c;
                raw.x[i][0] = *reinterpret_cast<const u4*>(t.kp + kw);
                if (m == 4) {
                    raw.x[i][1] = *reinterpret_cast<const u4*>(t.ks + 4 * km);
                    raw.x[i][2] = *reinterpret_cast<const u4*>(t.kz + 4 * km);
                } else {
                    const u2 ps = *reinterpret_cast<const u2*>(t.ks + 2 * km), pz = *reinterpret_cast<const u2*>(t.kz + 2 * km);
                    raw.x[i][1] = mf_u4{ps[0], ps[1], 0u, 0u};
                    raw.x[i][2] = mf_u4{pz[0], pz[1], 0u, 0u};
                }
            } else {
                const int c = min(32 * (u - DC) + 4 * vcq, D - 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int s = min(s0 + 4 * vtq + j, last);
                    raw.x[i][0][j] = t.vp[static_cast<size_t>(s) * a.Hkv * (D / 16) + (c >> 4)];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = min(s0 + 4 * vtq + j, last);
            const size_t vm = static_cast<size_t>(s) * a.Hkv;
            if (m == 4) {
                raw.vm[0][j] = *reinterpret_cast<const uint32_t*>(t.vs + 4 * vm);
                raw.vm[1][j] = *reinterpret_cast<const uint32_t*>(t.vz + 4 * vm);
            } else {
                raw.vm[0][j] = *reinterpret_cast<const uint16_t*>(t.vs + 2 * vm);
                raw.vm[1][j] = *reinterpret_cast<const uint16_t*>(t.vz + 2 * vm);
            }
            raw.ids[0][j] = *reinterpret_cast<const uint2*>(t.ids + min(s0 + 4 * ktq + j, last));
            raw.ids[1][j] = *reinterpret_cast<const uint2*>(t.ids + s);
        }
    };

    // Writes the fetched tile as f16 parts, masked tokens as zeros; the largest
    // key and value past the limit goes to `over`.
    auto stage = [&](const int tile, const float kscale, const float vscale, const bool first) {
        const bool packed = tile >= t.td;
        const int s0 = kTile * (tile - t.td), d0 = kTile * tile;
        bool kok[4], vok[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (packed) {
                kok[j] = s0 + 4 * ktq + j < t.slots && (raw.ids[0][j].x & raw.ids[0][j].y) != 0xffffffffu;
                vok[j] = s0 + 4 * vtq + j < t.slots && (raw.ids[1][j].x & raw.ids[1][j].y) != 0xffffffffu;
            } else {
                kok[j] = d0 + 4 * ktq + j < t.nd;
                vok[j] = d0 + 4 * vtq + j < t.nd;
            }
        }
        float vsc[4], vzr[4];
        if (packed) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                vsc[j] = a.meta_fp16 ? half_lo(raw.vm[0][j]) : __uint_as_float(raw.vm[0][j]);
                vzr[j] = a.meta_fp16 ? half_lo(raw.vm[1][j]) : __uint_as_float(raw.vm[1][j]);
            }
        }
        float kmx = 0.0f, vmx = 0.0f;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = wm + WM * i;
            if (u >= 2 * DC) break;
            const bool isk = u < DC;
            const int c0 = 32 * (isk ? u : u - DC) + 4 * (isk ? kcq : vcq);
            const bool in = c0 < D;  // channels past head_dim are zeros
            float x[4][4];  // [token][channel]
            if (!packed) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = __uint_as_float(raw.x[i][j][e]);
            } else if (isk) {
                float sc[4], zr[4];
                if (a.meta_fp16) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[e] = e & 1 ? half_hi(raw.x[i][1][e / 2]) : half_lo(raw.x[i][1][e / 2]);
                        zr[e] = e & 1 ? half_hi(raw.x[i][2][e / 2]) : half_lo(raw.x[i][2][e / 2]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[e] = __uint_as_float(raw.x[i][1][e]);
                        zr[e] = __uint_as_float(raw.x[i][2][e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = raw.x[i][0][e] >> (8 * (ktq & 3));  // codes of the lane's tokens in its low byte
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[j][e] = __builtin_fmaf(static_cast<float>((w >> (2 * j)) & 3u), sc[e], zr[e]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = raw.x[i][0][j] >> (8 * (vcq & 3));  // codes of the lane's channels
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[j][e] = __builtin_fmaf(static_cast<float>((w >> (2 * e)) & 3u), vsc[j], vzr[j]);
                }
            }
            if (isk) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[j][e] = (kok[j] && in) ? x[j][e] * kscale : 0.0f;
                        kmx = fmaxf(kmx, fabsf(x[j][e]));
                    }
                    const uint2 p = parts(x[j][0], x[j][1]), q = parts(x[j][2], x[j][3]);
                    char* d = tl + (4 * ktq + j) * L::KS + 2 * c0;
                    *reinterpret_cast<uint2*>(d + L::KHI) = make_uint2(p.x, q.x);
                    *reinterpret_cast<uint2*>(d + L::KLO) = make_uint2(p.y, q.y);
                }
            } else {
                // token quad vtq in the MFMA order: 8 tokens per lane group, its half by the 16-token tile
                const int kd = 16 * (vtq & 3) + 8 * (vtq >> 2);  // bytes
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        y[j] = (vok[j] && in) ? x[j][e] * vscale : 0.0f;
                        vmx = fmaxf(vmx, fabsf(y[j]));
                    }
                    const uint2 p = parts(y[0], y[1]), q = parts(y[2], y[3]);
                    char* d = tl + (c0 + e) * L::VS + kd;
                    *reinterpret_cast<uint2*>(d + L::VHI) = make_uint2(p.x, q.x);
                    *reinterpret_cast<uint2*>(d + L::VLO) = make_uint2(p.y, q.y);
                }
            }
        }
        if (wm == 0 && vcq == 0) {
            float* bias = reinterpret_cast<float*>(tl + L::BIAS) + 4 * vtq;
#pragma unroll
            for (int j = 0; j < 4; ++j) bias[j] = vok[j] ? 0.0f : kNegInf;
        }
        // (positive floats order like their bits)
        if (first) {
            if (kmx > 0.0f) atomicMax(reinterpret_cast<int*>(low), __float_as_int(kmx / kscale));
            if (vmx > 0.0f) atomicMax(reinterpret_cast<int*>(low) + 1, __float_as_int(vmx / vscale));
        }
        if (__ballot(kmx >= kLimit || vmx >= kLimit)) {
            // (an infinity has no exponent that helps: it makes NaN of what reads it)
            const float inf = __builtin_huge_valf();
            if (kmx >= kLimit && kmx < inf) atomicMax(reinterpret_cast<int*>(over), __float_as_int(fminf(kmx / kscale, 3.0e38f)));
            if (vmx >= kLimit && vmx < inf) atomicMax(reinterpret_cast<int*>(over) + 1, __float_as_int(fminf(vmx / vscale, 3.0e38f)));
        }
    };

    // Q' = Q 2^(12 - e), e the exponent of the row's largest value, as the QK B operand: row n of row tile rt, channels
    // 32 s + 8 g .. + 7.
    mf_u4 qh[RT][DC], ql[RT][DC];
    float crow[RT];  // log2 units per unit of the product
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = row0 + 16 * (RT * wm + rt) + n;
        const bool live = r < rows;
        const int seq = only >= 0 ? only : (live ? r / G : 0);
        const int h = kvh * G + (only >= 0 ? min(r, G - 1) : (live ? r % G : 0));
        const float* q = global_ptr(a.seqs[seq].Q) + static_cast<size_t>(h) * D;
        float x[DC][8];
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < DC; ++s) {
            const int c = 32 * s + 8 * g;
            typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = 0.0f;
            if (live && c < D) {
                const f4 y = *reinterpret_cast<const f4*>(q + c), z = *reinterpret_cast<const f4*>(q + c + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[s][j] = y[j];
                    x[s][4 + j] = z[j];
                }
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
    float mr[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        mr[rt] = -3.0e38f;
        l[rt] = 0.0f;
#pragma unroll
        for (int s = 0; s < 2 * DC; ++s) acc[rt][s] = mf_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int k_exp = 0, v_exp = 0;  // keys are staged as K 2^(4 - k_exp); uniform over the workgroup
    float* lrow = (only >= 0 && a.logits && a.seqs[only].mean_attn_weights)
                      ? a.logits + static_cast<size_t>(a.tok_base[only]) * a.Hq : nullptr;
    const int ld = lrow ? a.tok_base[only + 1] - a.tok_base[only] : 0;

    if (threadIdx.x < 4) over[threadIdx.x] = 0.0f;
    bool kfirst = true, vfirst = true;
    if (t0 + wt < t1) fetch(t0 + wt);
    for (int tb = t0; tb < t1; tb += WT) {
        const int tile = tb + wt;
        const bool mine = tile < t1;
        __syncthreads();  // the last tiles' readers are done
        if (mine)
            stage(tile, __builtin_amdgcn_ldexpf(16.0f, -k_exp), __builtin_amdgcn_ldexpf(16.0f, -v_exp), kfirst || vfirst);
        if (tile + WT < t1) fetch(tile + WT);
        __syncthreads();
        int k_new = k_exp, v_new = v_exp;
        if (kfirst || vfirst) {
            const float lk = low[0], lv = low[1];
            if (kfirst && __ballot(lk > 0.0f)) {
                kfirst = false;
                if (__ballot(lk < kLow)) k_new = scalar(__builtin_amdgcn_frexp_expf(lk)) - 11;
            }
            if (vfirst && __ballot(lv > 0.0f)) {
                vfirst = false;
                if (__ballot(lv < kLow)) v_new = scalar(__builtin_amdgcn_frexp_expf(lv)) - 11;
            }
        }
        const float ok = over[0], ov = over[1];
        if (__ballot(ok > 0.0f)) k_new = max(k_exp, scalar(__builtin_amdgcn_frexp_expf(ok)) - 11);
        if (__ballot(ov > 0.0f)) v_new = max(v_exp, scalar(__builtin_amdgcn_frexp_expf(ov)) - 11);
        if (k_new != k_exp || v_new != v_exp) {
            // keys or values outside what f16 holds well: new exponents, and the tiles again
            const float f = __builtin_amdgcn_ldexpf(1.0f, v_exp - v_new);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int s = 0; s < 2 * DC; ++s) acc[rt][s] *= f;
            k_exp = k_new;
            v_exp = v_new;
            __syncthreads();
            if (mine) {
                fetch(tile);
                stage(tile, __builtin_amdgcn_ldexpf(16.0f, -k_exp), __builtin_amdgcn_ldexpf(16.0f, -v_exp), false);
            }
            if (tile + WT < t1) fetch(tile + WT);
            __syncthreads();
            if (threadIdx.x < 2) over[threadIdx.x] = 0.0f;
        }
        if (!mine) continue;

        mf_f4 d[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 2; ++i) d[rt][i] = mf_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < DC; ++s) {
                const char* p = tl + (16 * i + n) * L::KS + 64 * s + 16 * g;
                const mf_u4 kh = *reinterpret_cast<const mf_u4*>(p + L::KHI);
                const mf_u4 kl = *reinterpret_cast<const mf_u4*>(p + L::KLO);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    d[rt][i] = mfma16x16x32(kh, ql[rt][s], d[rt][i]);
                    d[rt][i] = mfma16x16x32(kl, qh[rt][s], d[rt][i]);
                    d[rt][i] = mfma16x16x32(kh, qh[rt][s], d[rt][i]);
                }
            }
        mf_f4 bias[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) bias[i] = *reinterpret_cast<const mf_f4*>(tl + L::BIAS + 64 * i + 16 * g);
        mf_u4 ph[RT], pl[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float c = __builtin_amdgcn_ldexpf(crow[rt], k_exp);
            float s[2][4];
            float mx = kNegInf;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[i][r] = __builtin_fmaf(d[rt][i][r], c, bias[i][r]);
                    mx = fmaxf(mx, s[i][r]);
                }
            if (lrow) {
                const int r = row0 + 16 * (RT * wm + rt) + n;
                if (r < rows) {
                    const bool packed = tile >= t.td;
                    const int pos = packed ? t.nd + kTile * (tile - t.td) : kTile * tile;
                    const int end = packed ? t.nd + t.slots : t.nd;
                    float* o = lrow + static_cast<size_t>(kvh * G + r) * ld;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (pos + 16 * i + 4 * g + q < end) o[pos + 16 * i + 4 * g + q] = s[i][q];
                }
            }
            // the reference moves only when a row's maximum passes it by more than the slack
            if (__ballot(mx - kUp > mr[rt] + kSlack)) {
                mx = xrow_max(mx);
                const bool up = mx - kUp > mr[rt] + kSlack;
                const float mn = up ? mx - kUp : mr[rt];
                const float al = up ? __builtin_amdgcn_exp2f(mr[rt] - mn) : 1.0f;
                l[rt] *= al;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float ar = __shfl(al, 4 * g + r, 64);
#pragma unroll
                    for (int q = 0; q < 2 * DC; ++q) acc[rt][q][r] *= ar;
                }
                mr[rt] = mn;
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - mr[rt]);
                    sum += s[i][r];
                }
            l[rt] += sum;
            const uint2 p0 = parts(s[0][0], s[0][1]), p1 = parts(s[0][2], s[0][3]);
            const uint2 p2 = parts(s[1][0], s[1][1]), p3 = parts(s[1][2], s[1][3]);
            ph[rt] = mf_u4{p0.x, p1.x, p2.x, p3.x};
            pl[rt] = mf_u4{p0.y, p1.y, p2.y, p3.y};
        }
#pragma unroll
        for (int q = 0; q < 2 * DC; ++q) {
            const char* p = tl + (16 * q + n) * L::VS + 16 * g;
            const mf_u4 vh = *reinterpret_cast<const mf_u4*>(p + L::VHI);
            const mf_u4 vl = *reinterpret_cast<const mf_u4*>(p + L::VLO);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                acc[rt][q] = mfma16x16x32(pl[rt], vh, acc[rt][q]);
                acc[rt][q] = mfma16x16x32(ph[rt], vl, acc[rt][q]);
                acc[rt][q] = mfma16x16x32(ph[rt], vh, acc[rt][q]);
            }
        }
    }

    // A row's sum over its four lane groups; the partial in the units of V.
    const float vback = __builtin_amdgcn_ldexpf(1.0f, v_exp - 4);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = xrow_sum(l[rt]);
    auto partial = [&](const int r) {  // index of row r's partial
        const int seq = only >= 0 ? only : r / G;
        const int h = kvh * G + (only >= 0 ? r : r % G);
        const int ns = a.slot_base[seq + 1] - a.slot_base[seq];
        const int own = a.own_base[seq + 1] - a.own_base[seq];
        return static_cast<size_t>(a.slot_base[seq]) * a.Hq + static_cast<size_t>(h) * ns + (only >= 0 ? slot : own + slot);
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
                    if (16 * q < D) o[16 * q + n] = acc[rt][q][r] * vback;
            }
        }
    } else {
        // The waves of one row tile took other tokens: joined in LDS.
        constexpr int RW = 16 * RT;                 // rows of a wave
        constexpr int LINE = 32 * DC + 4;           // floats per row: accumulators, reference, sum
        static_assert(WM * WT * RW * LINE * 4 <= WT * L::BYTES, "the merge fits in the tiles' LDS");
        __syncthreads();
        float* my = reinterpret_cast<float*>(lds) + static_cast<size_t>(wave) * RW * LINE;
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
        __syncthreads();
        for (int idx = threadIdx.x; idx < WM * RW * 32 * DC; idx += 64 * WM * WT) {
            const int row = idx / (32 * DC), c = idx - row * 32 * DC;  // row of the workgroup, channel
            const int rr = row0 + row;
            if (rr >= rows || c >= D) continue;
            const float* x = reinterpret_cast<const float*>(lds) + static_cast<size_t>((row / RW) * RW + row % RW) * LINE;
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
            a.acc[pi * D + c] = A * vback;
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
// s % 8, back to back, so that a tile's lines come from memory once.
// OWN: the slots are the sequences' own, else the prefix's.
template <int DC, int RT, int WM, int WT, bool OWN>
__global__ void __launch_bounds__(64 * WM * WT) attn_shared_kernel(const SharedArgs a) {
    extern __shared__ __align__(16) char lds[];
    const unsigned id = blockIdx.x;
    const unsigned q = id >> 3;
    const unsigned hc = static_cast<unsigned>(a.Hkv * a.chunks);
    const int hz = static_cast<int>(q % hc);
    const int s = static_cast<int>((q / hc) * 8 + (id & 7));
    if (s >= a.total) return;
    const int kvh = hz / a.chunks, chunk = hz - kvh * a.chunks;
    const int G = a.Hq / a.Hkv;
    const int row0 = chunk * 16 * RT * WM;
    if constexpr (OWN) {
        const int i = find_seq(a.own_base, a.nseq, s);
        const int part = s - a.own_base[i], parts_ = a.own_base[i + 1] - a.own_base[i];
        const Tiers t = tiers_of(a.seqs[i], a, kvh);
        shared_body<DC, RT, WM, WT>(a, lds, t, kvh, row0, G, i, share(t.tiles, part, parts_),
                                    share(t.tiles, part + 1, parts_), part);
    } else {
        const Tiers t = tiers_of(a.prefix, a, kvh);
        shared_body<DC, RT, WM, WT>(a, lds, t, kvh, row0, a.nseq * G, -1, share(t.tiles, s, a.total),
                                    share(t.tiles, s + 1, a.total), s);
    }
}

template <int DC, int RT, int WM, int WT, bool OWN>
int launch(SharedArgs a, const int rows, hipStream_t st) {
    if (a.total <= 0) return TT_OK;
    a.chunks = (rows + 16 * RT * WM - 1) / (16 * RT * WM);
    const long long wgs = static_cast<long long>((a.total + 7) / 8) * 8 * a.Hkv * a.chunks;
    if (wgs > 0x00ffffffLL) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "attention grid too large");
    constexpr int bytes = WT * TileLds<DC>::BYTES + 16;
    const auto kernel = attn_shared_kernel<DC, RT, WM, WT, OWN>;
    TT_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(64 * WM * WT), bytes, st, a);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

// Rows per workgroup of the prefix: one 16-row tile with the waves along the
// tokens, or four waves of 16 or 32 rows on the same tokens.
constexpr int kFewRows = 16;

template <int DC>
int launch_dc(const SharedArgs& prefix, const SharedArgs& own, const int rows, const int G, hipStream_t st) {
    constexpr int WT = DC <= 4 ? 4 : 2;
    constexpr int RT = DC <= 4 ? 2 : 1;
    int rc = rows <= kFewRows ? launch<DC, 1, 1, WT, false>(prefix, rows, st) : launch<DC, RT, 4, 1, false>(prefix, rows, st);
    if (rc) return rc;
    return launch<DC, 1, 1, WT, true>(own, G, st);
}

}  // namespace

SharedPlan shared_plan(const tt_decode_seq& prefix, const tt_decode_seq* seqs, int nseq, int Hq, int Hkv, int D, int kgs) {
    SharedPlan p;
    BatchPlan& b = p.batch;
    b.nseq = nseq;
    const int G = Hq / Hkv, rows = nseq * G;
    auto tiles = [&](const tt_decode_seq& s) {
        return (static_cast<long long>(s.dense_count) + kTile - 1) / kTile +
               (static_cast<long long>(s.num_blocks) * kgs + kTile - 1) / kTile;
    };
    const int per_wg = rows <= kFewRows ? 16 : (D <= 128 ? 128 : 64);
    const long long heads = static_cast<long long>(Hkv) * ((rows + per_wg - 1) / per_wg);
    const long long pt = tiles(prefix);
    const long long waves_along = rows <= kFewRows ? (D <= 128 ? 4 : 2) : 1;
    if (pt > 0) p.prefix_slots = static_cast<int>(std::max<long long>(1, std::min({pt / waves_along, 512 / heads, 1024LL})));
    for (int i = 0; i < nseq; ++i) {
        const int n = static_cast<int>(std::max<long long>(1, std::min<long long>((tiles(seqs[i]) + 7) / 8, 1024)));
        b.pk_base[i + 1] = b.pk_base[i] + n;
        b.slot_base[i + 1] = b.slot_base[i] + n + p.prefix_slots;
    }
    batch_layout(b, seqs, Hq, D, kgs);
    return p;
}

int shared_launch(const SharedPlan& plan, const tt_decode_seq& prefix, const tt_decode_seq* seqs_dev, int Hq, int Hkv,
                  int D, int kgs, int meta_fp16, void* ws, hipStream_t stream) {
    const BatchPlan& b = plan.batch;
    char* base = static_cast<char*>(ws);
    SharedArgs a;
    a.seqs = seqs_dev;
    a.prefix = prefix;
    a.ml = reinterpret_cast<float*>(base + b.off_ml);
    a.acc = reinterpret_cast<float*>(base + b.off_acc);
    a.logits = reinterpret_cast<float*>(base + b.off_logits);
    a.scale2 = kLog2e / sqrtf(static_cast<float>(D));
    a.nseq = b.nseq;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    a.kgs = kgs;
    a.meta_fp16 = meta_fp16 ? 1 : 0;
    a.prefix_slots = plan.prefix_slots;
    a.chunks = 1;
    a.total = plan.prefix_slots;
    std::memcpy(a.slot_base, b.slot_base, sizeof(a.slot_base));
    std::memcpy(a.own_base, b.pk_base, sizeof(a.own_base));
    std::memcpy(a.tok_base, b.tok_base, sizeof(a.tok_base));
    SharedArgs own = a;
    own.total = b.pk_base[b.nseq];
    const int G = Hq / Hkv, rows = b.nseq * G;
    int rc;
    if (D <= 64)
        rc = launch_dc<2>(a, own, rows, G, stream);
    else if (D <= 96)
        rc = launch_dc<3>(a, own, rows, G, stream);
    else if (D <= 128)
        rc = launch_dc<4>(a, own, rows, G, stream);
    else if (D <= 192)
        rc = launch_dc<6>(a, own, rows, G, stream);
    else
        rc = launch_dc<8>(a, own, rows, G, stream);
    if (rc) return rc;
    return batch_finalize(b, seqs_dev, Hq, D, kgs, ws, stream);
}

}  // namespace tt
