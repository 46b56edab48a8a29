// What the kernels of the generation operators are given (cache.cu,
// sampling.cu, prefix_attention.cu); generation.cpp checks the tensors and
// fills these in.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace mnb {

namespace cache {

// A page pool seen as [planes][pages][page_chunks] 16-byte chunks.
struct Pool {
  void* base;
  long long plane_chunks;
  int page_chunks, token_chunks, planes, pages, page_size;
};

struct Table {
  int* table;  // [slots][columns], row stride ld
  int* lens;   // [slots]
  int* refs;   // [pages]
  long long ld;
  int slots, columns, pages, page_size;
};

struct Append {
  __nv_bfloat16 *k_pool, *v_pool;
  long long page_ld, token_ld, head_ld;
  const __nv_bfloat16 *k, *v;
  long long k_ld, k_head, v_ld, v_head;
  const int* table;
  long long table_ld;
  int slots, columns, pages, page_size;
  const int* positions;
  const int* slot_of;  // or null: token i belongs to row i
  int n, heads, chunks;
};

cudaError_t launch_copy(const Pool& p, int* src, int* dst, int* tokens, int* count, int n, int* status, cudaStream_t stream);
// scratch: 4 n + slots ints
cudaError_t launch_fork(const Pool& p, const Table& t, const int* parents, const int* children, int n, int* scratch,
                        int* status, cudaStream_t stream);
// scratch: pages + n + slots ints
cudaError_t launch_reserve(const Table& t, const int* slots, const int* counts, int n, int* scratch, int* status,
                           cudaStream_t stream);
cudaError_t launch_free(const Table& t, const int* slots, int n, int* status, cudaStream_t stream);
// scratch: 3 pages + 1 ints
constexpr int kSmallTable = 16 * 1024;  // entries that the planning block remaps itself, in less time than a launch takes
cudaError_t launch_compact(const Pool& p, const int* table, long long table_ld, int rows, int columns, const int* refs,
                           int* new_table, int* new_refs, int* scratch, int* status, cudaStream_t stream);
cudaError_t launch_append(const Append& a, int* status, cudaStream_t stream);

}  // namespace cache

namespace sampling {

constexpr int kIndexBits = 20;  // a vocabulary has at most 2^20 tokens

struct Setting {
  const float* each;
  float all;
};
struct WholeSetting {
  const int* each;
  int all;
};

struct Sample {
  const void* logits;
  bool bf16;
  long long ld;
  const float* noise;
  long long noise_ld;
  int rows, vocab;
  Setting temperature;
  WholeSetting top_k;
  Setting top_p, min_p;
  long long* token;
  float* logprob;  // or null
  int* status;
};

cudaError_t launch_sample(const Sample& a, cudaStream_t stream);

}  // namespace sampling

namespace prefix {

struct Args {
  const __nv_bfloat16* q;
  long long q_ld, q_head;
  const __nv_bfloat16 *k, *v;
  long long page_ld, token_ld, head_ld;  // of the page pools, in elements
  int pages, page_shift;
  int no_page;  // an index outside the pool's tensor map, where TMA reads zeros: for ids that name no page
  const int* prefix_pages;
  int prefix_len;
  const int* page_table;
  long long table_ld;
  const int* seq_lens;
  const int* q_offsets;  // or null: one row for each sequence
  int n, batch, kv_heads, group, heads;
  int max_q, max_len;
  float scale_log2;  // the scores' factor times log2(e)
  // the pieces (plan)
  bool tensor_cores;  // the prefix by prefix_attention_tc.cu
  int tile_rows;      // rows that a block of the other kernel takes at once
  bool quad;          // it takes four kv heads of a sequence at once
  int row_tiles, prefix_splits, prefix_chunk;
  int own_tiles, own_splits, own_chunk;
  float* part_o;    // [pieces][n][heads][head_dim]
  float2* part_ml;  // [pieces][n][heads]: maximum (log2 units) and sum
  int* sound;  // or null, without q_offsets: whether they give every row to one sequence; if not, the rows of the own
               // keys' pieces are in part unwritten, and nobody reads them
  __nv_bfloat16* o;
  float* lse;  // or null
  int* status;  // of waits
  int* errors;  // of bad indices
};

#ifdef __CUDACC__
// Whether the partial results of own keys count, for a kernel behind those that write them.  (The word comes by way of L1:
// fetched from L2 by every warp of the join, it made 16 x 512 tokens of 16 heads of 64 7 % slower.)
__device__ __forceinline__ bool own_count(const Args& a) { return !a.sound || *a.sound != 0; }
#endif

// Splits the keys into pieces; returns how many partial results each row gets.
int plan(Args& a, int head_dim);
// head dims 64 and 128; with one prefix piece, joins the rows and finishes them
cudaError_t launch_prefix_tc(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, int head_dim, cudaStream_t stream);
// the tensor-core kernel's own 2^x, on 2 * pairs numbers
cudaError_t launch_exp2(const float* x, float* y, int pairs, cudaStream_t stream);
cudaError_t launch_attention(const Args& a, int head_dim, cudaStream_t stream);
int kernels(const Args& a);  // that launch_attention() launches

}  // namespace prefix

}  // namespace mnb
