// attention.cuh — attention over a paged KV pool whose requests share a prefix
// (see attention.cu).
#pragma once

#include "common.cuh"

namespace gsec {

struct AttnArgs {
  const char* q;            // [tokens, hq, dim]; byte strides of a token and of a head
  int64_t q_pitch, q_head;
  int64_t tokens;
  int hq, hk, group, dim;   // group = hq / hk
  const char* pool;         // slot records: pitch bytes, V at + plane
  int64_t pitch, plane, pool_rows;
  const int32_t* cu;        // [batch + 1] query offsets
  const int32_t* lens;      // [batch] own keys of a request (its new tokens among them)
  int batch;
  const int32_t* table;     // [batch, width] pages, row pitch in elements
  int64_t table_pitch;
  int width, page;
  FastDiv page_div, group_div;
  const int32_t* prefix;    // pages of the shared prefix
  int32_t prefix_len;
  float scale;
  char* out;                // [tokens, hq, dim]
  float* lse;               // [tokens, hq] or null
  char* workspace;
};

int64_t attention_workspace(const AttnArgs& a, int dtype);
int attention(const AttnArgs& a, int dtype, cudaStream_t s);
// Bit 0: a page outside the pool, or lengths that do not fit the batch; bit 1: a bounded wait gave up.
unsigned attention_device_status(bool clear);

}  // namespace gsec
