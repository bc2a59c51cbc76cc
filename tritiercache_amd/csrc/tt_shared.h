// tt_shared.h -- host interface of the shared-prefix decode attention (tt_shared.hip).
#pragma once
#include "tt_attn.h"

namespace tt {

// Split-K plan of a launch over seqs[0, batch.nseq) behind one prefix. The
// partial slots of sequence i are the run slot_base[i] .. slot_base[i + 1] of
// the batched plan's layout: its own slots first, then prefix_slots slots that
// the prefix kernel fills for every query head of the sequence.
struct SharedPlan {
    BatchPlan batch;             // pk_base: prefix of the sequences' own slots
    int prefix_slots = 0;        // 0: no prefix tokens
};

SharedPlan shared_plan(const tt_decode_seq& prefix, const tt_decode_seq* seqs, int nseq, int Hq, int Hkv, int D, int kgs);
// Enqueues the partials of the prefix and of the sequences' own tiers, and the
// batched merge / mean weights.
int shared_launch(const SharedPlan& plan, const tt_decode_seq& prefix, const tt_decode_seq* seqs_dev, int Hq, int Hkv,
                  int D, int kgs, int meta_fp16, void* ws, hipStream_t stream);

}  // namespace tt
