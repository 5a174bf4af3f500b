/*
 * lf_ragged_params.h — parameter blocks of the kernels for sequences and requests of different lengths, for C and C++ hosts
 * that launch them through lf_shim.h: the device structs of loopfuse_amd/csrc/kernels restated with fixed-width host types,
 * field for field.  loopfuse_amd/packed.py and loopfuse_amd/paged.py hold the ctypes mirrors and fill them; a C host finds
 * there what each field is computed from.  Pointers are device pointers; strides are in elements where nothing else is said.
 */
#ifndef LF_RAGGED_PARAMS_H
#define LF_RAGGED_PARAMS_H

#include "lf_attn_params.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A tile of a packed batch, an entry of the lists that lf_packed_plan writes. */
typedef struct LfPackedTileHost {
  int32_t row0;            /* first row of the sequence */
  int32_t len;             /* its rows; 0: no tile */
  int32_t tile;            /* number of the tile in it */
  int32_t seq;             /* number of the sequence; -1: rows of no sequence */
} LfPackedTileHost;

/* lf_packed_sort, then lf_packed_plan: the lists of a packed batch, for tiles of 32, 64, 128 and 256 rows, each for sequences
 * in groups of 1, 2, 4 and 8: list (height i, group size j) begins at entry 4 * (cap[0] + ... + cap[i-1]) + j * cap[i]. */
typedef struct LfPackedPlanParamsHost {
  const int32_t* offsets;  /* [N + 1] */
  LfPackedTileHost* tiles; /* [4 * (cap[0] + ... + cap[3])] */
  int32_t* sorted;         /* scratch, [7][N + 2] */
  int32_t N, T;            /* sequences, 2^22 at most; rows, 2^31 - 1024 at most */
  int32_t cap[4];          /* entries of a list: T / height + N + 2 */
} LfPackedPlanParamsHost;

/* lf_attn_prefill_swp -DLF_PACKED=1: B = 1, Sq = Sk = T, *_sb unused, part_ml optional [Hq, T]. */
typedef struct LfPackedAttnParamsHost {
  LfAttnParamsHost attn;
  const LfPackedTileHost* tiles;   /* a list for tiles of 128 rows (128 / g with -DLF_GQAPACK=g) */
  void* low;               /* optional, shape and strides of O: what rounding took from O, for a backward */
  int32_t clear;           /* 1: zeros into rows of no sequence */
} LfPackedAttnParamsHost;

/* The backward kernels with -DLF_PACKED=1: B = 1, Sq = Sk = T, lse and delta [Hq, T]; rows of Q, K, V and dO lie D elements apart or more
 * (what is read behind a sequence's last row has to lie outside it). */
typedef struct LfPackedBwdParamsHost {
  LfAttnBwdParamsHost bwd;
  const LfPackedTileHost* dkdv_tiles;      /* lists for tiles of as many keys, and queries, as a workgroup has */
  const LfPackedTileHost* dq_tiles;
  const void* low;         /* optional, strides of O: as the forward wrote it */
  int32_t dkdv_blocks;     /* lf_attn_bwd_both (-DLF_BW_BOTH=1): workgroups of dK and dV, in front of those of dQ */
} LfPackedBwdParamsHost;

/* lf_attn_decode -DLF_SHARED=1, then lf_shared_combine.  attn: q_sb, q_sh, q_ss = request, kv head, row of its group, o likewise;
 * Sk = keys of the prefix, nsplit and split_len those of its splits; part_acc [pieces, Hkv, rows, D], part_ml [pieces, Hkv, rows, 2]
 * with room for 2^target_log2 / units + B pieces of own keys. */
typedef struct LfSharedParamsHost {
  LfAttnParamsHost attn;
  const int32_t* lengths;  /* [B] own keys of each request */
  const void* prefix_k;    /* page ids of the prefix, of the tables' type */
  const void* prefix_v;
  float* pre_acc;          /* [Hkv, nsplit, B * rows, D], 16-byte aligned as part_acc */
  float* pre_ml;           /* [Hkv, nsplit, B * rows, 2] */
  int32_t room;            /* own keys that a row of the tables has room for, 2^30 at most */
  int32_t units;           /* workgroups per piece of own keys */
  int32_t pre_units;       /* workgroups per split of the prefix ... */
  int32_t pre_blocks;      /* ... and in all */
  int32_t target_log2;     /* workgroups that the own keys are cut for */
  int32_t least;           /* least length of a piece, a multiple of 32 */
} LfSharedParamsHost;

/* lf_paged_tables */
typedef struct LfTablesParamsHost {
  const int32_t* cached;   /* [B] */
  const int32_t* fresh;    /* [B] new tokens */
  void* table;             /* [B, width], int32 or int64 (LF_TABLE_I64) */
  const void* free;        /* [count], likewise */
  int32_t* offsets;        /* [B + 1] */
  int32_t* lengths;        /* [B] */
  int32_t* slots;          /* [T] */
  int32_t* positions;      /* [T] */
  int32_t* pages;          /* [1] */
  int64_t table_stride;
  int32_t B, width, count, T;
  int32_t shift;           /* log2 of the tokens per page */
} LfTablesParamsHost;

/* lf_store_kv */
typedef struct LfStoreParamsHost {
  const void* k;           /* [T, heads, 8 * per_head] */
  const void* v;
  void* k_pool;            /* [pages, page, heads, 8 * per_head] */
  void* v_pool;
  const int32_t* slots;    /* [T]; below 0 or `last` and more: left out */
  int64_t k_ss, k_sh, v_ss, v_sh;                    /* strides in pieces of 16 bytes: rows, heads */
  int64_t kp_sb, kp_ss, kp_sh, vp_sb, vp_ss, vp_sh;  /* pages, tokens of a page, heads */
  int64_t last;            /* slots of a pool */
  int32_t T, heads, per_head;      /* T: 2^31 - 256 at most */
  int32_t shift;           /* log2 of the tokens per page */
} LfStoreParamsHost;

#ifdef __cplusplus
}
#endif

#endif /* LF_RAGGED_PARAMS_H */
