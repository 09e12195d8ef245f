// The routing's interface to the mixture-of-experts layer.
#pragma once

#include <stdio.h>

#include "common.h"
#include "qwen4mix_internal.h"

// The logits of a call: x [rows, hidden] (rows ldx apart) against the router
// [experts, hidden] and, where shared_router is given, one more column for it;
// logits [rows, cols], cols = experts (+ 1).
template <typename T>
struct QmLogits {
  const T* x;
  long ldx;
  const T* router;
  const T* shared_router;
  double* logits;
  int rows, hidden, experts, cols;
  int* counts;         // [experts + 1] cleared with the logits, or null
};

// float words of the scratch that qm_route needs beside the logits, in bytes
size_t qm_route_norms(int rows, int experts);

// The logits of a few rows, summed in double (one launch).
template <typename T> int qm_route_logits(const QmLogits<T>& A, hipStream_t stream);

// What the choice leaves for the experts' products: each expert's pairs (pair
// ppt t + j is choice j of token t) in counts and lists [experts][rows], and the
// table of row tiles, (grid row, first row) of every tile of bm rows: grid row y is
// shared expert y or expert y - shared. counts holds one word more.
struct QmRouteLists {
  int* counts;
  int* lists;
  int* n_tiles;
  int2* tiles;
  int ppt, shared, bm;
};

// Logits and choice (two launches): ids [rows, top_k], weights [rows, ld_w] of the
// choices and, behind them, `shared` times the sigmoid of the last column (or 1);
// with `lists`, those too.
template <typename T>
int qm_route(const QmLogits<T>& A, int top_k, int normalize, int* ids, float* weights, int ld_w, int shared,
             const QmRouteLists* lists, float* norms, hipStream_t stream);

// The argument checks that the two entry points share.
int qm_check_route(const char* what, int act_dtype, int rows, int hidden, int experts, int top_k, long ldx);
