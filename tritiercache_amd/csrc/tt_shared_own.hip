// tt_shared_own.hip -- partials of the sequences' own tiers behind a shared
// prefix, for all sequences in one launch (gfx950): the matrix-core loop of the
// batched decode for head_dim 128, the VALU loop for every other one. A short
// prefix of few sequences is read here too, once per sequence.
#include "tt_shared.h"
#include "tt_attn_dev.h"
#include "tt_attn_line.h"

#include <algorithm>

namespace tt {
namespace {

constexpr int kOwnTileCost = 4;  // 16 FP32 tokens in pairs of 16 packed ones, as in the batch's plan

struct OwnArgs {
    const tt_decode_seq* __restrict__ seqs;
    tt_decode_seq prefix;
    float* ml;
    float* acc;
    float* logits;
    float scale2;
    int entries, per_seq, total_slots, Hq, Hkv, D, kgs, meta_fp16, hc, chunks;
    int slot_base[kMaxBatchSeqs + 1];  // runs of the sequences
    int tok_base[kMaxBatchSeqs + 1];
    int pk_base[kMaxBatchSeqs + 1];    // packed slots of the entries, then
    int dn_base[kMaxBatchSeqs + 1];    // their FP32 ones
};

// The prefix's or the sequence's pointer, in scalar registers: of a choice the
// compiler would otherwise make a load from a chosen address.
template <typename T>
__device__ __forceinline__ T* pick(const bool pre, T* x, T* y) {
    const uint64_t a = reinterpret_cast<uint64_t>(x), b = reinterpret_cast<uint64_t>(y);
    const uint32_t lo = pre ? static_cast<uint32_t>(a) : static_cast<uint32_t>(b);
    const uint32_t hi = pre ? static_cast<uint32_t>(a >> 32) : static_cast<uint32_t>(b >> 32);
    return global_ptr<T>(static_cast<uint64_t>(static_cast<uint32_t>(scalar(static_cast<int>(hi)))) << 32 |
                         static_cast<uint32_t>(scalar(static_cast<int>(lo))));
}

// The arguments of entry e, a sequence's own tiers or (odd e of two) the
// prefix's for its query; the prefix has no logits, and its slots lie behind
// the own ones in the sequence's run.
__device__ __forceinline__ SplitArgs entry_args(const OwnArgs& b, const int e) {
    const int i = scalar(b.per_seq == 2 ? e >> 1 : e);
    const bool pre = b.per_seq == 2 && (e & 1);
    const tt_decode_seq& s = b.seqs[i];
    SplitArgs a;
    a.in.Q = global_ptr(s.Q);
    a.in.k0 = pick(pre, b.prefix.dense_K, s.dense_K);
    a.in.v0 = pick(pre, b.prefix.dense_V, s.dense_V);
    a.in.n0 = scalar(pre ? b.prefix.dense_count : s.dense_count);
    a.in.kp = pick(pre, b.prefix.PBS_K_Packed, s.PBS_K_Packed);
    a.in.ks = pick(pre, b.prefix.PBS_K_Scales, s.PBS_K_Scales);
    a.in.kz = pick(pre, b.prefix.PBS_K_Zeroes, s.PBS_K_Zeroes);
    a.in.vp = pick(pre, b.prefix.PBS_V_Packed, s.PBS_V_Packed);
    a.in.vs = pick(pre, b.prefix.PBS_V_Scales, s.PBS_V_Scales);
    a.in.vz = pick(pre, b.prefix.PBS_V_Zeroes, s.PBS_V_Zeroes);
    a.in.ids = pick(pre, b.prefix.PBS_token_ids, s.PBS_token_ids);
    a.in.num_blocks = scalar(pre ? b.prefix.num_blocks : s.num_blocks);
    a.in.Hq = b.Hq;
    a.in.Hkv = b.Hkv;
    a.in.D = b.D;
    a.in.kgs = b.kgs;
    a.in.meta_fp16 = b.meta_fp16;
    a.scale2 = b.scale2;
    const int own = pre ? b.pk_base[e] - b.pk_base[e - 1] + b.dn_base[e] - b.dn_base[e - 1] : 0;  // slots before these
    a.part_ml = b.ml + static_cast<size_t>(b.slot_base[i]) * b.Hq * 2 + 2 * own;
    a.part_acc = b.acc + static_cast<size_t>(b.slot_base[i]) * b.Hq * b.D + static_cast<size_t>(own) * b.D;
    a.logits = !pre && s.mean_attn_weights ? b.logits + static_cast<size_t>(b.tok_base[i]) * b.Hq : nullptr;
    a.ld = b.tok_base[i + 1] - b.tok_base[i];
    a.nsplit = b.slot_base[i + 1] - b.slot_base[i];
    a.nsplit_p = b.pk_base[e + 1] - b.pk_base[e];
    a.nsplit_d = b.dn_base[e + 1] - b.dn_base[e];
    a.dense_delay = 0;
    return a;
}

// head_dim 128: grid and slots as the batched decode's (attn_batched_kernel).
template <int GP, typename MetaT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(GP == 8 ? 3 : 1)))
attn_own_kernel(const OwnArgs b) {
    constexpr int kLds = MfLds<GP>::TOTAL > DnLds<GP>::TOTAL ? MfLds<GP>::TOTAL : DnLds<GP>::TOTAL;
    __shared__ __align__(16) char lds[kLds];
    const unsigned id = blockIdx.x;
    const unsigned q = id >> 3;
    const int hz = static_cast<int>(q % static_cast<unsigned>(b.hc));
    const int g = static_cast<int>((q / static_cast<unsigned>(b.hc)) * 8 + (id & 7));
    if (g >= b.total_slots) return;
    const int npk = b.pk_base[b.entries];
    int e, s;
    if (g < npk) {
        e = batch_find(b.pk_base, b.entries, g);
        s = g - b.pk_base[e];
    } else {
        e = batch_find(b.dn_base, b.entries, g - npk);
        s = (b.pk_base[e + 1] - b.pk_base[e]) + (g - npk - b.dn_base[e]);
    }
    const SplitArgs a = entry_args(b, e);
    const int kvh = hz / b.chunks, chunk = hz - kvh * b.chunks;
    if (s >= a.nsplit_p) {
        dense_body<GP>(a, s - a.nsplit_p, kvh, chunk, lds);
        return;
    }
    packed_body<GP, MetaT, false, true>(a, s, kvh, chunk, lds);
}

// Every other head_dim: grid (slots, KV heads, head chunks), both kinds of
// tiers in a slot (pk_base counts them, dn_base is all zeros).
template <int CPL, int GP, typename MetaT>
__global__ void __launch_bounds__(256) attn_own_split_kernel(const OwnArgs b) {
    __shared__ __align__(16) char lds[SplitLds<CPL, GP>::BYTES];
    const int g = static_cast<int>(blockIdx.x);
    if (g >= b.total_slots) return;
    const int e = batch_find(b.pk_base, b.entries, g);
    SplitArgs a = entry_args(b, e);
    a.nsplit_d = a.nsplit_p;
    a.nsplit_p = 0;
    split_body<CPL, GP, MetaT, true>(a, g - b.pk_base[e], lds);
}

template <int GP>
int launch_own_mfma(const OwnArgs& b, hipStream_t st) {
    const long long wgs = static_cast<long long>((b.total_slots + 7) / 8) * 8 * b.hc;
    if (wgs > 0x00ffffffLL) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "attention grid too large");
    const dim3 grid(static_cast<unsigned>(wgs));
    if (b.meta_fp16)
        hipLaunchKernelGGL((attn_own_kernel<GP, uint16_t>), grid, dim3(256), 0, st, b);
    else
        hipLaunchKernelGGL((attn_own_kernel<GP, float>), grid, dim3(256), 0, st, b);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

template <int CPL, int GP>
int launch_own_split(const OwnArgs& b, hipStream_t st) {
    const long long slots = (static_cast<long long>(b.total_slots) + 7) / 8 * 8;  // slot s of every head on XCD s % 8
    if (slots * b.hc > 0x00ffffffLL || b.Hkv > 65535) TT_FAIL(TT_ERR_INVALID_ARGUMENT, "attention grid too large");
    const dim3 grid(static_cast<unsigned>(slots), b.Hkv, b.chunks);
    if (b.meta_fp16)
        hipLaunchKernelGGL((attn_own_split_kernel<CPL, GP, uint16_t>), grid, dim3(256), 0, st, b);
    else
        hipLaunchKernelGGL((attn_own_split_kernel<CPL, GP, float>), grid, dim3(256), 0, st, b);
    TT_LAUNCH_CHECK();
    return TT_OK;
}

template <int CPL>
int launch_own_split_g(const OwnArgs& b, const int gp, hipStream_t st) {
    switch (gp) {
    case 1: return launch_own_split<CPL, 1>(b, st);
    case 2: return launch_own_split<CPL, 2>(b, st);
    case 4: return launch_own_split<CPL, 4>(b, st);
    default: return launch_own_split<CPL, 8>(b, st);
    }
}

}  // namespace

BatchPlan own_plan(const tt_decode_seq* entries, int n, int per_seq, int Hq, int Hkv, int D, int kgs, int meta_fp16) {
    if (use_packed_kernel(D)) {
        if (per_seq == 1) return batch_plan(entries, n, Hq, Hkv, D, kgs, meta_fp16);
        // The batch's plan fills the device once, with eight units (a pair of packed 16-token words each) or more per slot.
        // Where the prefix is read with many sequences, their few own tokens take most of that, and each prefix is left to
        // a slot: then three rounds, every slot with about as much to do (24 sequences behind 4k, 28/4 heads: 64.8 ->
        // 34.2 us, 16 behind 4k, 32/8 heads: 56.6 -> 34.7; 8 behind 8k, which are left to the batch's plan, 32.1 | 33.0).
        // And where there is little to do, slots of four units (2 sequences behind 580, 32/8 heads: 13.3 -> 11.7 us, 1
        // behind 2048 14.0 -> 12.6; 8 behind 580 13.5 | 16.8).
        BatchPlan p;
        p.nseq = n;
        auto pairs = [&](const int i) { return (static_cast<long long>(entries[i].num_blocks) * (kgs / 16) + 1) / 2; };
        auto tiles = [&](const int i) { return (static_cast<long long>(entries[i].dense_count) + 15) / 16; };
        long long total = 0;
        for (int i = 0; i < n; ++i) total += pairs(i) + kOwnTileCost * tiles(i);
        const int heads = n / 2 * head_chunks(Hq, Hkv);
        const long long budget = std::max<long long>(1, 3LL * 256 / head_chunks(Hq, Hkv));
        const bool little = heads <= 32 && total < 8 * budget;
        if (!little && heads <= 64) return batch_plan(entries, n, Hq, Hkv, D, kgs, meta_fp16);
        const long long cap = std::max<long long>(little ? 4 : 16, (total + budget - 1) / budget);
        for (int i = 0; i < n; ++i) {
            const int np = static_cast<int>(std::max<long long>(1, (pairs(i) + cap - 1) / cap));
            const int nd = static_cast<int>((kOwnTileCost * tiles(i) + cap - 1) / cap);
            p.pk_base[i + 1] = p.pk_base[i] + np;
            p.dn_base[i + 1] = p.dn_base[i] + nd;
            p.slot_base[i + 1] = p.slot_base[i] + np + nd;
        }
        p.total_slots = p.slot_base[n];
        return p;
    }
    // The VALU loop: units of its kind per slot so that all slots make about two rounds of three workgroups per CU, at
    // least one unit for each of a slot's four waves.
    BatchPlan p;
    p.nseq = n;
    const int unit = split_unit_tokens(D);
    auto units = [&](const int i) {
        return (static_cast<long long>(entries[i].dense_count) + unit - 1) / unit +
               static_cast<long long>(entries[i].num_blocks) * (kgs / 16);
    };
    long long total = 0;
    for (int i = 0; i < n; ++i) total += units(i);
    const long long budget = std::max<long long>(1, 2LL * 3 * 256 / head_chunks(Hq, Hkv));
    const long long cap = std::max<long long>(4, (total + budget - 1) / budget);
    for (int i = 0; i < n; ++i) {
        const int s = static_cast<int>(std::max<long long>(1, (units(i) + cap - 1) / cap));
        p.pk_base[i + 1] = p.pk_base[i] + s;
        p.slot_base[i + 1] = p.slot_base[i] + s;
    }
    p.total_slots = p.slot_base[n];
    return p;
}

int own_launch(const SharedPlan& plan, const tt_decode_seq& prefix, const tt_decode_seq* seqs_dev, int Hq, int Hkv,
               int D, int kgs, int meta_fp16, void* ws, hipStream_t stream) {
    const BatchPlan& b = plan.batch;
    char* base = static_cast<char*>(ws);
    const int gp = gp_for(Hq / Hkv);
    OwnArgs a;
    a.seqs = seqs_dev;
    a.prefix = prefix;
    a.ml = reinterpret_cast<float*>(base + b.off_ml);
    a.acc = reinterpret_cast<float*>(base + b.off_acc);
    a.logits = reinterpret_cast<float*>(base + b.off_logits);
    a.scale2 = kLog2e / sqrtf(static_cast<float>(D));
    a.entries = plan.entries.nseq;
    a.per_seq = plan.per_seq;
    a.total_slots = plan.entries.total_slots;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.D = D;
    a.kgs = kgs;
    a.meta_fp16 = meta_fp16 ? 1 : 0;
    a.chunks = (Hq / Hkv + gp - 1) / gp;
    a.hc = Hkv * a.chunks;
    std::memcpy(a.slot_base, b.slot_base, sizeof(a.slot_base));
    std::memcpy(a.tok_base, b.tok_base, sizeof(a.tok_base));
    std::memcpy(a.pk_base, plan.entries.pk_base, sizeof(a.pk_base));
    std::memcpy(a.dn_base, plan.entries.dn_base, sizeof(a.dn_base));
    if (use_packed_kernel(D)) {
        switch (gp) {
        case 1: return launch_own_mfma<1>(a, stream);
        case 2: return launch_own_mfma<2>(a, stream);
        case 4: return launch_own_mfma<4>(a, stream);
        default: return launch_own_mfma<8>(a, stream);
        }
    }
    switch (D / 16) {
    case 1: return launch_own_split_g<1>(a, gp, stream);
    case 2: return launch_own_split_g<2>(a, gp, stream);
    case 3: return launch_own_split_g<3>(a, gp, stream);
    case 4: return launch_own_split_g<4>(a, gp, stream);
    case 5: return launch_own_split_g<5>(a, gp, stream);
    case 6: return launch_own_split_g<6>(a, gp, stream);
    case 7: return launch_own_split_g<7>(a, gp, stream);
    case 9: return launch_own_split_g<9>(a, gp, stream);
    case 10: return launch_own_split_g<10>(a, gp, stream);
    case 11: return launch_own_split_g<11>(a, gp, stream);
    case 12: return launch_own_split_g<12>(a, gp, stream);
    case 13: return launch_own_split_g<13>(a, gp, stream);
    case 14: return launch_own_split_g<14>(a, gp, stream);
    case 15: return launch_own_split_g<15>(a, gp, stream);
    default: return launch_own_split_g<16>(a, gp, stream);
    }
}

}  // namespace tt
