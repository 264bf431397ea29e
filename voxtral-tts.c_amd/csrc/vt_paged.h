/*
 * vt_paged.h - the handle of a batch over a paged cache, shared by what writes pages (vt_paged.hip) and what reads them (vt_paged_attention.hip).
 */
#ifndef VT_PAGED_H
#define VT_PAGED_H

#include "vt_state.h"
#include "vt_paged_plans.h"

struct tts_hip_paged {
    vt_paged_shape shape;
    int max_seqs, max_rows, max_table, max_items;
    int device;                          /* that the buffers below are on; -1: none yet */
    /* one block each: positions | places | tables | items, at the same offsets; `described`: the most that comes before the items */
    unsigned char *host, *dev;
    size_t at_place, at_tables, at_items, described, bytes;
    hipEvent_t copied;                   /* the last batch has left `host` */
    int *starts, *written;
    unsigned long long *seen;            /* a bit for each page, 0 between calls */
    /* the batch, and how it is worked on; n_seqs -1: none yet */
    int n_seqs, n_rows;
    vt_paged_plan plan[2];               /* for fp32 and bf16 queries */
    int bf16_items;                      /* the second one's first item */
};

int vt_paged_ready(const char *who, const tts_hip_paged *b);      /* a batch of this context's device; else an error */

#endif /* VT_PAGED_H */
