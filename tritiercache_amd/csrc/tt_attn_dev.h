// tt_attn_dev.h -- device code of the decode attention partials (the kernels
// around it are in tt_attn.hip and tt_shared_own.hip): the matrix-core loop over
// the packed store (tt_attn_mfma.h) and the VALU loop.
#pragma once
#include "tt_attn.h"
#include "tt_wave.h"

namespace tt {
namespace {

template <int N>
__device__ __forceinline__ void load_f32(const float* __restrict__ p, float (&x)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + j);
            x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 v = *reinterpret_cast<const float2*>(p + j);
            x[j] = v.x; x[j + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = p[j];
    }
}

// The FP32 tiers' addresses as values in scalar registers: a per-lane choice
// between them is then a select. (Left to the compiler it becomes a load of the
// chosen pointer from the kernel arguments, a round trip before each tile's
// own loads.)
struct TierPtrs {
    uint64_t k0, k1, k2, v0, v1, v2;
};
__device__ __forceinline__ TierPtrs tier_ptrs(const AttnInputs& in) {
    auto u = [](const float* p) { return reinterpret_cast<uint64_t>(p); };
    TierPtrs t{u(in.k0), u(in.k1), u(in.k2), u(in.v0), u(in.v1), u(in.v2)};
    asm("" : "+s"(t.k0), "+s"(t.k1), "+s"(t.k2), "+s"(t.v0), "+s"(t.v1), "+s"(t.v2));
    return t;
}
__device__ __forceinline__ const float* global_f32(const uint64_t a) { return global_ptr<const float>(a); }

struct SplitArgs {
    AttnInputs in;
    float scale2;  // log2(e) / sqrt(head_dim): logits are kept in log2 units
    float* part_ml;
    float* part_acc;
    float* logits;
    int ld;
    int nsplit;      // partial slots per query head
    int nsplit_p;    // matrix-core workgroups over the packed store: slots [0, nsplit_p)
    int nsplit_d;    // VALU workgroups: slots [nsplit_p, nsplit)
    int dense_delay; // FP32-tier workgroups wait this many 10 ns ticks before their first tile load
};

#include "tt_attn_mfma.h"

// Largest i < n with base[i] <= x (base non-decreasing, base[0] = 0 <= x).
__device__ __forceinline__ int batch_find(const int* base, const int n, const int x) {
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

// ---------------------------------------------------------------------------
// The VALU loop (head_dim other than 128, 64 with an odd number of KV heads,
// and short contexts of both). FP32 arithmetic throughout: operands, products
// and sums.
// ---------------------------------------------------------------------------

// Tokens of one FP32 unit of a wave: half a tile for the head dims whose rows of four tokens per lane would take
// 128 registers.
__host__ __device__ constexpr int split_unit_tokens(const int D) { return D > 128 ? 8 : 16; }

// Floats of one (value, row group) line in the merge area: 16 channel lanes and one of padding.
constexpr int kSplitLine = 17;

// LDS of the VALU tile loop: per wave the accumulators and the sums of its
// heads, reduced over the wave's row groups, and its maxima.
template <int CPL, int GP>
struct SplitLds {
    static constexpr int VALUES = (GP * (CPL + 1) + 3) / 4 * 4;  // GP x CPL accumulators, GP sums, padding
    static constexpr int BYTES = 4 * (VALUES * kSplitLine + GP) * 4;
};

// N consecutive words, floats or metadata entries in as few loads as their
// count allows. They need be aligned to an entry only (a head's row starts at
// a multiple of head_dim entries, a lane's slice at a multiple of head_dim /
// 16): the types say two bytes, and the hardware takes any.
template <int N>
__device__ __forceinline__ void load_slice(const uint32_t* __restrict__ p, uint32_t (&x)[N]) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
    typedef uint32_t u1 __attribute__((aligned(2)));
    constexpr int N4 = N / 4 * 4;
#pragma unroll
    for (int j = 0; j < N4; j += 4) {
        const u4 v = *reinterpret_cast<const u4*>(p + j);
        x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
    }
    if constexpr (N - N4 >= 2) {
        const u2 v = *reinterpret_cast<const u2*>(p + N4);
        x[N4] = v.x; x[N4 + 1] = v.y;
    }
    if constexpr ((N - N4) % 2 == 1) x[N - 1] = *reinterpret_cast<const u1*>(p + N - 1);
}
template <int N>
__device__ __forceinline__ void load_slice(const float* __restrict__ p, float (&x)[N]) {
    uint32_t u[N];
    load_slice<N>(reinterpret_cast<const uint32_t*>(p), u);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __uint_as_float(u[j]);
}
// Metadata of a lane's slice in its stored width, converted where it is used.
template <typename MetaT, int N>
struct MetaSlice;
template <int N>
struct MetaSlice<float, N> {
    float v[N];
    __device__ __forceinline__ void load(const float* __restrict__ p) { load_slice<N>(p, v); }
    __device__ __forceinline__ float get(const int j) const { return v[j]; }
};
template <int N>
struct MetaSlice<uint16_t, N> {
    static constexpr bool kPairs = N % 2 == 0;  // read two entries per word
    uint32_t v[kPairs ? N / 2 : N];
    __device__ __forceinline__ void load(const uint16_t* __restrict__ p) {
        if constexpr (kPairs) {
            load_slice<N / 2>(reinterpret_cast<const uint32_t*>(p), v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = p[j];
        }
    }
    __device__ __forceinline__ float get(const int j) const {
        if constexpr (kPairs)
            return f16_to_f32(static_cast<uint16_t>((j & 1) ? v[j / 2] >> 16 : v[j / 2] & 0xffffu));
        else
            return f16_to_f32(static_cast<uint16_t>(v[j]));
    }
};

__device__ __forceinline__ float meta_value(const float v) { return v; }
__device__ __forceinline__ float meta_value(const uint16_t v) { return f16_to_f32(v); }

// The codes at bits 0, 8, 16 and 24 of x, each alone in its byte, from where
// one conversion makes a float of it. (Opaque, or the compiler extracts every
// code with an instruction of its own and converts it from byte 0.)
__device__ __forceinline__ uint32_t code_bytes(const uint32_t x) {
    uint32_t y = x & 0x03030303u;
    asm("" : "+v"(y));
    return y;
}

// Sum over the four 16-lane rows of four values at once: row r of the result
// holds the total of v[r] (two swaps that exchange half of the rows, an add
// after each).
__device__ __forceinline__ float rows_sum4(const float (&v)[4]) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[2]), __float_as_uint(v[3]), false, false);
    const float x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const float y = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// CPL: channels per lane (head_dim / 16). GP: query heads per workgroup
// (padded to a power of two; heads past the group repeat its last one and are
// never stored).
//
// Each wave owns a contiguous share of its KV head's units: FP32 units of
// split_unit_tokens, then 16-token packed tiles, counted alike (an FP32 unit
// holds more bytes and needs fewer instructions; at two, four or eight tiles
// per FP32 unit the launches took the same or up to 15% longer). Wave w of
// workgroup `split` has share w nsplit_d + split, so that every workgroup
// holds both kinds. Lane (row group tg, channel lane cp) holds channels cp CPL
// .. + CPL - 1 of tokens tg, tg + 4, ...: a K word shifted by 2 tg has those
// tokens' codes in the low bits of its four bytes, so one mask and four byte
// conversions unpack them. The row's logits come from a DPP sum over its 16
// lanes; V is unpacked after the softmax, when K is no longer live.
//
// A wave has one to three units, so the launch is a chain: arguments, query
// and first unit's loads, arithmetic (about 850 VALU instructions per packed
// tile at head_dim 256 with two heads, 350 at head_dim 80 with one), the next
// unit, the merge. What it responds to is the length of that chain: 32-bit
// shares of the work (64-bit divides took about 2 us), loads as wide as the
// row allows from scalar bases, and registers for as many waves per SIMD as the
// heads of a group leave (seven at head_dim 64 with one head, three at 128 with
// four, two at 128 and one at 256 with eight).
// Partials per launch: head_dim 256 with 16/8 heads at 8k 18.7 -> 11.6 us,
// head_dim 80 with 32/32 heads at 2k 10.3 -> 6.2, head_dim 96 with 32/32
// heads at 4k 15.2 -> 9.1, head_dim 64 with 9/3 heads at 8k 9.4 -> 6.4.
//
// CLEAN: the V scale and zero of masked slots count as zeros, whatever they
// are (else a NaN or an infinity there makes a NaN of its zero weight).
template <int CPL, int GP, typename MetaT, bool CLEAN = false>
__device__ __forceinline__ void split_body(const SplitArgs& a, const int split, char* lds) {
    constexpr int D = 16 * CPL;
    constexpr int NTD = split_unit_tokens(D) / 4;  // FP32 tokens per lane and unit
    const AttnInputs& in = a.in;
    const int kvh = blockIdx.y;
    const int G = in.Hq / in.Hkv;
    const int g0 = blockIdx.z * GP;
    const int gc = min(GP, G - g0);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tg = lane >> 4;
    const int cp = lane & 15;

    float q[GP][CPL];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
        // heads past the group repeat its last one (their results are not stored)
        load_slice<CPL>(in.Q + static_cast<size_t>(kvh * G + g0 + min(g, gc - 1)) * D + cp * CPL, q[g]);
    }

    int n0 = in.n0, n1 = in.n1, n2 = in.n2, head = in.ring_head, nb = in.num_blocks;
    if (in.state) {
        n0 = scalar(in.state[kSCount]);
        n1 = scalar(in.state[kHhCount]);
        n2 = scalar(in.state[kRwCount]);
        head = scalar(in.state[kRwHead]);
        nb = scalar(in.state[kBlocksUsed]);
    }
    const int Nd = n0 + n1 + n2;
    const int W = in.kgs >> 4;
    const int Td = (Nd + 4 * NTD - 1) / (4 * NTD);
    const int Tp = nb * W;
    const int Hkv = in.Hkv;

    // The wave's share of the Td FP32 units and Tp packed tiles.
    const int part = wave * a.nsplit_d + split, parts = 4 * a.nsplit_d;
    const int lo = part_begin(Td + Tp, part, parts), hi = part_begin(Td + Tp, part + 1, parts);
    const int d_begin = min(lo, Td), d_end = min(hi, Td);
    const int p_begin = max(lo - Td, 0), p_end = max(hi - Td, 0);

    float m[GP], l[GP], acc[GP][CPL];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
        m[g] = kNegInf;
        l[g] = 0.0f;
#pragma unroll
        for (int j = 0; j < CPL; ++j) acc[g][j] = 0.0f;
    }

    // Lane cp = NT (g % HS) + i stores the logit of head g, token tok0 + tg + 4 i.
    auto put_logits = [&](const auto& s, const int tok0, const int limit) {
        constexpr int NT = sizeof(s) / sizeof(s[0]);
        constexpr int HS = 16 / NT < GP ? 16 / NT : GP;  // heads per store
#pragma unroll
        for (int h0 = 0; h0 < GP; h0 += HS) {
            float v = s[0][h0];
#pragma unroll
            for (int g = 0; g < HS; ++g)
#pragma unroll
                for (int i = 0; i < NT; ++i) v = (cp == NT * g + i) ? s[i][h0 + g] : v;
            const int g = h0 + cp / NT, t = tok0 + tg + 4 * (cp % NT);
            if (cp < NT * HS && g < gc && t < limit)
                st_dev1(a.logits + static_cast<size_t>(kvh * G + g0 + g) * a.ld + t, v);
        }
    };
    // Online softmax: logits to weights, the accumulators to the new maximum
    // (exact, and the same in every lane).
    auto softmax = [&](auto& s) {
        constexpr int NT = sizeof(s) / sizeof(s[0]);
#pragma unroll
        for (int g = 0; g < GP; ++g) {
            float tm = s[0][g];
#pragma unroll
            for (int i = 1; i < NT; ++i) tm = fmax_nn(tm, s[i][g]);
            const float mn = fmax_nn(m[g], xrow_max(tm));
            const float alpha = (m[g] == kNegInf) ? 0.0f : __builtin_amdgcn_exp2f(m[g] - mn);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                s[i][g] = (s[i][g] == kNegInf) ? 0.0f : __builtin_amdgcn_exp2f(s[i][g] - mn);
                sum += s[i][g];
            }
            l[g] = __builtin_fmaf(l[g], alpha, sum);
#pragma unroll
            for (int j = 0; j < CPL; ++j) acc[g][j] *= alpha;
            m[g] = mn;
        }
    };

    const TierPtrs tier = tier_ptrs(in);
#pragma unroll 1
    for (int k = d_begin; k < d_end; ++k) {
        // ---- FP32 unit: logical rows 4 NTD k ... ----
        const int tok0 = 4 * NTD * k;
        float kx[NTD][CPL], vx[NTD][CPL];
        // (V's addresses up to head_dim 128 at once, from byte offsets, which takes up to ten registers less than a base
        // and an offset each; above, where two waves per SIMD are planned for, the latter is 0.1 to 0.3 us faster.)
        constexpr bool kBytes = D <= 128;
        size_t off[NTD];
        uint64_t vb[NTD];
#pragma unroll
        for (int i = 0; i < NTD; ++i) {
            const int r = min(tok0 + tg + 4 * i, Nd - 1);  // rows past the tiers are masked below
            const bool in0 = r < n0, in1 = r < n0 + n1;
            int ring = head + (r - n0 - n1);
            ring = ring >= in.ring_size ? ring - in.ring_size : ring;
            const int idx = in0 ? r : (in1 ? r - n0 : ring);
            off[i] = (static_cast<size_t>(idx) * Hkv + kvh) * D + cp * CPL;
            const uint64_t kb = in0 ? tier.k0 : (in1 ? tier.k1 : tier.k2);
            vb[i] = in0 ? tier.v0 : (in1 ? tier.v1 : tier.v2);
            if constexpr (kBytes) {
                const uint64_t bytes = sizeof(float) * off[i];
                vb[i] += bytes;
                load_slice<CPL>(global_f32(kb + bytes), kx[i]);
            } else {
                load_slice<CPL>(global_f32(kb) + off[i], kx[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NTD; ++i) load_slice<CPL>(global_f32(vb[i]) + (kBytes ? 0 : off[i]), vx[i]);
        float s[NTD][GP];
#pragma unroll
        for (int i = 0; i < NTD; ++i)
#pragma unroll
            for (int g = 0; g < GP; ++g) {
                float d = 0.0f;
#pragma unroll
                for (int j = 0; j < CPL; ++j) d = __builtin_fmaf(q[g][j], kx[i][j], d);
                d = row_sum16(d) * a.scale2;
                s[i][g] = (tok0 + tg + 4 * i < Nd) ? d : kNegInf;
            }
        if (a.logits) put_logits(s, tok0, Nd);
        softmax(s);
        // Rows past the tiers repeat the last one, whose V may be infinite: a
        // zero weight alone would make a NaN of it.
        if (tok0 + 4 * NTD > Nd) {
#pragma unroll
            for (int i = 0; i < NTD; ++i)
#pragma unroll
                for (int j = 0; j < CPL; ++j) vx[i][j] = (tok0 + tg + 4 * i < Nd) ? vx[i][j] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NTD; ++i)
#pragma unroll
            for (int g = 0; g < GP; ++g)
#pragma unroll
                for (int j = 0; j < CPL; ++j) acc[g][j] = __builtin_fmaf(s[i][g], vx[i][j], acc[g][j]);
    }

    const MetaT* ks = static_cast<const MetaT*>(in.ks);
    const MetaT* kz = static_cast<const MetaT*>(in.kz);
    const MetaT* vs = static_cast<const MetaT*>(in.vs);
    const MetaT* vz = static_cast<const MetaT*>(in.vz);
    // The lane's CPL channels are 2 CPL bits of the row's code words, from bit
    // 2 (c0 % 16) of word c0 / 16 on (in two words where CPL does not divide 16).
    constexpr bool kOneWord = (16 % CPL) == 0;
    const int c0 = cp * CPL;
    const int cw = c0 >> 4, csh = 2 * (c0 & 15);
    const int cw1 = min(cw + 1, CPL - 1);
    // Loads take a wave-uniform base and a 32-bit lane offset: K words and
    // metadata from the tile's (block's) row, V words and metadata from the
    // rows of tokens 4 i, at the same lane offset for every i. (The offset is
    // opaque, or its 64-bit extension is hoisted out of the loop and every
    // load takes a 64-bit vector add instead of the scalar base.)
    auto at = [](const void* base, uint32_t off) {
        asm("" : "+v"(off));
        return static_cast<const char*>(base) + off;
    };
    const uint32_t k_off = static_cast<uint32_t>(kvh * D + c0);
    const uint32_t v_row = static_cast<uint32_t>(tg * Hkv + kvh);
    const uint32_t v_off = (v_row * CPL + cw) * 4u, v_off1 = (v_row * CPL + cw1) * 4u;

#pragma unroll 1
    for (int t = p_begin; t < p_end; ++t) {
        // ---- 2-bit packed tile: half (kgs 32) or whole (kgs 16) block ----
        // (an opaque copy of the index: the compiler would keep an address per
        // load in registers over the loop, about 30 in all)
        int kt = t;
        asm("" : "+s"(kt));
        const size_t krow = static_cast<size_t>(kt) * Hkv * D;
        const size_t mrow = static_cast<size_t>(W == 2 ? kt >> 1 : kt) * Hkv * D;
        const size_t slot0 = static_cast<size_t>(16) * kt;
        const long long id = *reinterpret_cast<const long long*>(at(in.ids + slot0, 8u * cp));
        uint32_t kw[CPL];
        MetaSlice<MetaT, CPL> ksc, kze;
        load_slice<CPL>(reinterpret_cast<const uint32_t*>(at(in.kp + krow, 4u * k_off)), kw);
        ksc.load(reinterpret_cast<const MetaT*>(at(ks + mrow, sizeof(MetaT) * k_off)));
        kze.load(reinterpret_cast<const MetaT*>(at(kz + mrow, sizeof(MetaT) * k_off)));
        uint32_t vw[4], vw1[4];
        MetaT vsr[4], vzr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t row = (slot0 + 4 * i) * Hkv;
            vw[i] = *reinterpret_cast<const uint32_t*>(at(in.vp + row * CPL, v_off));
            vw1[i] = kOneWord ? 0u : *reinterpret_cast<const uint32_t*>(at(in.vp + row * CPL, v_off1));
            vsr[i] = *reinterpret_cast<const MetaT*>(at(vs + row, sizeof(MetaT) * v_row));
            vzr[i] = *reinterpret_cast<const MetaT*>(at(vz + row, sizeof(MetaT) * v_row));
        }
        float s[4][GP];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int g = 0; g < GP; ++g) s[i][g] = 0.0f;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const uint32_t x = code_bytes(kw[j] >> (2 * tg));
            const float sc = ksc.get(j), ze = kze.get(j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float kd = __builtin_fmaf(static_cast<float>((x >> (8 * i)) & 0xffu), sc, ze);
#pragma unroll
                for (int g = 0; g < GP; ++g) s[i][g] = __builtin_fmaf(q[g][j], kd, s[i][g]);
            }
        }
        const unsigned valid = static_cast<unsigned>(__ballot(id != -1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool ok = (valid >> (tg + 4 * i)) & 1u;
#pragma unroll
            for (int g = 0; g < GP; ++g) {
                const float d = row_sum16(s[i][g]) * a.scale2;
                s[i][g] = ok ? d : kNegInf;
            }
        }
        if (a.logits) put_logits(s, Nd + 16 * kt, Nd + 16 * kt + 16);
        softmax(s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = kOneWord ? vw[i] >> csh : __builtin_amdgcn_alignbit(vw1[i], vw[i], csh);
            const bool seen = !CLEAN || ((valid >> (tg + 4 * i)) & 1u);
            const float vsc = seen ? meta_value(vsr[i]) : 0.0f, vze = seen ? meta_value(vzr[i]) : 0.0f;
            // channel 4 b + k in byte b of word k (fewer than eight channels: the codes one by one)
            uint32_t wk[4];
            if constexpr (CPL >= 8) {
#pragma unroll
                for (int k = 0; k < 4; ++k) wk[k] = code_bytes(w >> (2 * k));
            }
#pragma unroll
            for (int j = 0; j < CPL; ++j) {
                const uint32_t c = CPL >= 8 ? (wk[j & 3] >> (8 * (j >> 2))) & 0xffu : (w >> (2 * j)) & 3u;
                const float v = __builtin_fmaf(static_cast<float>(c), vsc, vze);
#pragma unroll
                for (int g = 0; g < GP; ++g) acc[g][j] = __builtin_fmaf(s[i][g], v, acc[g][j]);
            }
        }
    }

    // Reduce the four row groups (each accumulated its own tokens), four
    // values at a time, then merge the four waves in LDS and store one partial
    // per query head.
    constexpr int NV = SplitLds<CPL, GP>::VALUES;
    float* sm = reinterpret_cast<float*>(lds);  // [4 waves][NV][kSplitLine]
    float* sm_m = sm + 4 * NV * kSplitLine;     // [4][GP]
    auto value = [&](const int v) {
        return v < GP * CPL ? acc[v / CPL][v % CPL] : (v < GP * (CPL + 1) ? l[v - GP * CPL] : 0.0f);
    };
#pragma unroll
    for (int v = 0; v < NV; v += 4) {
        const float x[4] = {value(v), value(v + 1), value(v + 2), value(v + 3)};
        sm[(wave * NV + v + tg) * kSplitLine + cp] = rows_sum4(x);
    }
    if (lane == 0) {
#pragma unroll
        for (int g = 0; g < GP; ++g) sm_m[wave * GP + g] = m[g];
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < gc * D; idx += 256) {
        const int g = idx / D, c = idx - g * D;
        const int line = g * CPL + c % CPL, col = c / CPL;
        float M = kNegInf;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w * GP + g]);
        float A = 0.0f, L = 0.0f;
        if (M != kNegInf) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float mw = sm_m[w * GP + g];
                const float f = (mw == kNegInf) ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
                A = __builtin_fmaf(f, sm[(w * NV + line) * kSplitLine + col], A);
                L = __builtin_fmaf(f, sm[(w * NV + GP * CPL + g) * kSplitLine], L);
            }
        }
        const size_t pi = static_cast<size_t>(kvh * G + g0 + g) * a.nsplit + a.nsplit_p + split;
        st_dev1(a.part_acc + pi * D + c, A);
        if (c == 0) {
            st_dev1(a.part_ml + 2 * pi, M);
            st_dev1(a.part_ml + 2 * pi + 1, L);
        }
    }
}

}  // namespace
}  // namespace tt
