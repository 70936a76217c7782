// Entry points of expert_sort.cu: slots (token, choice) of a router's decisions ordered by expert, rows copied there and back.
#pragma once

#define CCF_SORT_MAX_EXPERTS 1024
#define CCF_SORT_MAX_ALIGN 65536
#define CCF_SORT_MAX_SLOTS (1LL << 30)
#define CCF_SORT_MAX_D (1LL << 24)

#ifdef __cplusplus
extern "C" {
#endif

// Slots are numbered token-major. Rows of expert e begin at base[e], a multiple of `align`.
typedef struct CcfOrder {
  const void* idx;     // [slots] expert of each slot; outside [0, experts): none
  int* slot_row;       // [slots] row of each slot, -1: none
  int* row_slot;       // [rows] slot of each row, -1: none
  int* counts;         // [experts] rows of each expert
  int* base;           // [experts + 1]
  void* scratch;       // ccf_order_scratch bytes
  long long slots, rows, capacity;   // rows = ccf_order_rows; capacity: most rows of one expert
  int experts, align, wide, pad0;    // wide: idx is int64
} CcfOrder;

// Rows of tokens [tokens, d] and of sorted rows [rows, d] (contiguous).
typedef struct CcfRows {
  const void* tokens_in;   // [tokens, d], rows `ld` apart
  const void* rows_in;     // [rows, d]
  void* tokens_out;        // [tokens, d]
  void* rows_out;          // [rows, d]
  const int* slot_row;     // [tokens, top_k]
  const int* row_slot;     // [rows]
  const void* weights;     // [tokens, top_k] or null
  void* d_weights;         // [tokens, top_k]
  long long tokens, rows, ld;
  int top_k, d, type, weight_type;   // elements.cuh's types
} CcfRows;

int ccf_sizeof_order();
int ccf_sizeof_rows();
long long ccf_order_rows(long long slots, int experts, long long capacity, int align);   // -1: arguments out of range
long long ccf_order_scratch(long long slots, int experts);
// launches made, or a negative code
int ccf_order(const CcfOrder* o, void* stream);
// rows_out[slot_row[t, j]] = tokens_in[t], zeros in rows without a slot. `behind_order`: right behind ccf_order on the same stream, which nothing but it
// wrote row numbers for
int ccf_sort_rows(const CcfRows* r, int behind_order, void* stream);
// Both, `r` with the order's slot_row and row_slot; launches made, or a negative code
int ccf_sort_by_expert(const CcfOrder* o, const CcfRows* r, void* stream);
// tokens_out[t] = sum over j of weights[t, j] * rows_in[slot_row[t, j]]; without weights, of the rows alone
int ccf_return_rows(const CcfRows* r, void* stream);
// its gradients: rows_out[slot_row[t, j]] = weights[t, j] * tokens_in[t], zeros elsewhere; d_weights[t, j] = <tokens_in[t], rows_in[slot_row[t, j]]>.
// Either output may be null.
int ccf_return_rows_bwd(const CcfRows* r, void* stream);

#ifdef __cplusplus
}
#endif
