// tt_shared.h -- host interface of the shared-prefix decode attention
// (tt_shared.hip: the prefix for all sequences at once; tt_shared_own.hip: each
// sequence's own tiers).
#pragma once
#include "tt_attn.h"

namespace tt {

// Split-K plan of a launch over seqs[0, batch.nseq) behind one prefix. The
// partial slots of sequence i are the run batch.slot_base[i] ..
// batch.slot_base[i + 1], which the batched merge reads: the slots of its
// entries, then prefix_slots slots that the prefix kernel fills for every query
// head. A sequence has one entry, its own tiers, or two (per_seq = 2): its own
// and the prefix's, read for this sequence alone.
struct SharedPlan {
    BatchPlan batch;
    BatchPlan entries;       // slots of each entry (pk_base: packed, or of both kinds; dn_base: FP32)
    int per_seq = 1;
    int prefix_slots = 0;    // of which the first packed_slots share the packed tiles, the others the FP32 ones
    int packed_slots = 0;
    bool lone = false;       // a slot is one wave's, not a workgroup's
};

SharedPlan shared_plan(const tt_decode_seq& prefix, const tt_decode_seq* seqs, int nseq, int Hq, int Hkv, int D, int kgs,
                       int meta_fp16);
// Enqueues the partials of the prefix and of the entries, and the batched merge / mean weights.
int shared_launch(const SharedPlan& plan, const tt_decode_seq& prefix, const tt_decode_seq* seqs_dev, int Hq, int Hkv,
                  int D, int kgs, int meta_fp16, void* ws, hipStream_t stream);

// Slots of `n` entries (at most kMaxBatchSeqs), per_seq of each sequence, and the launch that fills them.
BatchPlan own_plan(const tt_decode_seq* entries, int n, int per_seq, int Hq, int Hkv, int D, int kgs, int meta_fp16);
int own_launch(const SharedPlan& plan, const tt_decode_seq& prefix, const tt_decode_seq* seqs_dev, int Hq, int Hkv,
               int D, int kgs, int meta_fp16, void* ws, hipStream_t stream);

}  // namespace tt
