// Kernel argument blocks and host-side launchers (one per kernel file).
#pragma once
#include "atf_common.h"

namespace atf {

// Prefill geometry (the oracle's tile quantization is block_m = kPfRowsWave
// query positions by block_n = kPfWinN keys).  8 waves of 32 rows: at most 256
// registers per wave, so two waves share each SIMD and one wave's softmax
// overlaps the other's MFMAs.
constexpr int kPfWaves = 8;
constexpr int kPfRowsWave = 32;
constexpr int kPfRowsWg = kPfWaves * kPfRowsWave;
constexpr int kPfTileN = 64;
constexpr int kPfWinN = 32;

// Decode geometry (block_n = one page).
constexpr int kDecMaxGroup = 16;
constexpr int kDecUnroll = 4;      // pages in flight per wave
constexpr int kDecWaves = 8;       // waves per workgroup (one split), 2 per SIMD
constexpr int kDecWavesShort = 4;  // the same for contexts too short to give 256 splits of 8 waves
constexpr int kDecMaxSplits = 256;
constexpr int kDecChipWaves = 2048;  // waves of a decode that the chip holds: two per SIMD
// Fixed device scratch of the entry point that allocates nothing
// (atf_decode_paged_bf16_noalloc): split partials, laid out as in a workspace.
constexpr size_t kDecScratchBytes = size_t(8) << 20;

struct KvWriteArgs {
  uint16_t* kv_cache;  // [num_pages][hkv][V half | K half]
  int num_pages, hkv;
  const uint16_t* k_src;
  const uint16_t* v_src;
  int64_t ks_b, ks_t, ks_h, vs_b, vs_t, vs_h;
  int batch, n_tokens;
  const int32_t* start_pos;  // [batch], absolute position of source token 0
  const int32_t* page_table;
  int max_pages;
  const float* rope_cs;
  int rope_max_pos;
  int layout;
  // Packed rows: sequence b's tokens are rows cu_tokens[b] .. cu_tokens[b + 1] - 1 of
  // k_src and v_src (total_tokens rows), at most n_tokens of them; null: row t of
  // sequence b lies at b ks_b + t ks_t.
  const int32_t* cu_tokens;
  int total_tokens;
  // Packed rows into pages of their own (start_pos and page_table are not read): row i of
  // sequence b goes to page cu_tokens[b] / 16 + b + i / 16, which is entered here.
  int32_t* own_table;
  int8_t* kv_exps;  // the 8-bit cache's exponents [num_pages][hkv][2] (kv_cache: its codes)
  int page_round;   // 8-bit writer: pages that are dealt out to the XCDs together
};

// The rows of sequence b in a call: the first, relative to k_src's and v_src's row 0
// of the sequence (strides ks_b, vs_b), and how many.
struct KvRows {
  int64_t first;
  int count;
};
template <bool kPacked>
__device__ __forceinline__ int kv_start(const KvWriteArgs& a, int b) {
  return kPacked && a.own_table != nullptr ? 0 : a.start_pos[b];
}
// The page of entry `pidx` of sequence b, and in a call with pages of its own its entry.
template <bool kPacked>
__device__ __forceinline__ int kv_page(const KvWriteArgs& a, const KvRows& rows, int b, int64_t pidx, bool enter) {
  const int64_t at = static_cast<int64_t>(b) * a.max_pages + pidx;
  if (!kPacked || a.own_table == nullptr) return a.page_table[at];
  const int pg = static_cast<int>(rows.first / kPage + b + pidx);
  if (enter) a.own_table[at] = pg;
  return pg;
}
template <bool kPacked>
__device__ __forceinline__ KvRows kv_rows(const KvWriteArgs& a, int b) {
  if (!kPacked) return KvRows{0, a.n_tokens};
  const int lo = max(a.cu_tokens[b], 0), hi = min(max(a.cu_tokens[b + 1], 0), a.total_tokens);  // (hi - lo: 32 bits)
  return KvRows{lo, max(0, min(hi - lo, a.n_tokens))};
}

// Queries of several sequences packed one after the other.
struct PackedRows {
  const int32_t* cu;        // [batch + 1] first rows
  const int32_t* seq_lens;  // [batch] keys, the sequence's queries the last of them; null: as many as queries
  int total_q;              // rows of q, out and lse
  int max_k;                // keys of a sequence at most
  const int32_t* tiles;     // launch_prefill_plan's list (null: not needed)
};

struct PrefillArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;
  uint16_t* out;
  int64_t o_sb, o_st, o_sh;
  float* lse;  // [B][Hq][nq] natural-log LSE, or null
  const uint16_t* kv_cache;  // [num_pages][hkv][V half | K half]
  int num_pages;
  const int32_t* page_table;
  int max_pages;
  int batch, nq, nk, q_offset, hq, hkv, group;
  int n_qtiles;  // set by launch_prefill for the kernel it picks
  float scale_log2;
  float sm_scale;
  const float* rope_cs;
  int layout;
  LevelTable lt;
  PackedRows pk;  // prefill_packed kernels (nq, nk, q_offset, q_sb and o_sb unused there)
};

struct DecodeArgs {
  const uint16_t* q;  // [B][Hq][128] (strided)
  int64_t q_sb, q_sh;
  uint16_t* out;  // [B][Hq][128] (strided)
  int64_t o_sb, o_sh;
  const uint16_t* kv_cache;  // [num_pages][hkv][V half | K half]; the 8-bit decode's codes
  const int8_t* kv_exps;     // 8-bit decode: [num_pages][hkv][2], V's and K's exponent
  int num_pages;
  const int32_t* page_table;
  int max_pages;
  const int32_t* seq_lens;
  int max_seq_len;
  int batch, hq, hkv, group;
  int n_splits, pages_per_split;
  int waves;  // kDecWaves or kDecWavesShort per workgroup
  bool spread;     // one workgroup per wave of a split (decode_wave_kernel); waves = kDecWaves
  bool by_length;  // with spread: the longest sequences' waves first
  float scale_log2;
  const float* rope_cs;
  int layout;
  // Window.  per_key = 0: the level table lt, page rule (block_n = 16): every
  // key of a page reads the 2 L levels' slices of its youngest key, L >= 1.
  // per_key = 1: the per-slice (vec8) table st, slice s of a key at age z read
  // iff z <= st.zhi[s] (the FlashInfer port's rule, no minimum).
  LevelTable lt;
  SliceTable st;
  int per_key;
  // partials: of splits (n_splits > 1), or with spread of the splits' waves
  float* ws_ml;        // [B][Hkv][n_splits][16][2],   [B][Hkv][n_splits][8][2][group]
  float* ws_o;         // [B][Hkv][n_splits][16][128], [B][Hkv][n_splits][8][group][128]
};

// K and V of a contiguous decode: rows [batch][token][head][128] (element strides).
struct DecodeRows {
  const uint16_t* k;
  const uint16_t* v;
  int64_t ks_b, ks_t, ks_h, vs_b, vs_t, vs_h;
};

// Block tables and slot maps of a step's new tokens (atf_extend_tables).
constexpr int kTabMaxBatch = 8191;  // sequences: two prefix sums in 64 KB of LDS
struct ExtendTablesArgs {
  int32_t* page_table;
  int max_pages;
  const int32_t* seq_lens;
  const int32_t* new_lens;
  const int32_t* free_pages;
  int num_free;
  const int32_t* free_count;
  int batch, total, num_pages;
  int32_t* lens_out;
  int32_t* free_left;
  int32_t* cu_out;
  int32_t* positions;
  int64_t* slots;
};
hipError_t launch_extend_tables(const ExtendTablesArgs& a, hipStream_t s);
struct ReleaseTablesArgs {
  int32_t* page_table;
  int max_pages;
  int32_t* seq_lens;
  int32_t* free_pages;
  int num_free;
  int32_t* free_count;
  const int32_t* rows;
  int n_rows, batch, num_pages;
};
hipError_t launch_release_tables(const ReleaseTablesArgs& a, hipStream_t s);

hipError_t launch_kv_write(const KvWriteArgs& a, hipStream_t s);
// The writer of the 8-bit cache.
hipError_t launch_kv_write_q8(const KvWriteArgs& a, hipStream_t s);
// Blocks of the 8-bit cache -> blocks of a bf16 cache: entry (b, p), p < n_pages, of the
// page table to block b n_pages + p of `out`, that number (or -1 for an entry outside
// the pool, whose block is left as it is) to out_table[b][p].  out_table null: page g to
// block g of `out`, which has num_pages of them.
struct KvExpandArgs {
  const uint8_t* codes;
  const int8_t* exps;
  int num_pages, hkv;
  const int32_t* page_table;
  int batch, max_pages, n_pages;
  const int32_t* seq_lens;  // tokens of each sequence (null: n_pages pages of each); -1 for entries past them
  uint16_t* out;
  int32_t* out_table;
};
hipError_t launch_kv_expand_q8(const KvExpandArgs& a, hipStream_t s);
hipError_t launch_prefill(const PrefillArgs& a, hipStream_t s);
// Packed rows: the list of query tiles (prefill_plan_bytes, 0 where none is needed; a.pk,
// batch and heads are read), then the attention over it.
size_t prefill_plan_bytes(int batch, int total_q, int hq);
hipError_t launch_prefill_plan(const PrefillArgs& a, int32_t* tiles, hipStream_t s);
hipError_t launch_prefill_packed(const PrefillArgs& a, hipStream_t s);
// The MFMA-ceiling probe of the prefill (measurement only): sink holds
// ceil(ceil(nq / 256) / 8) * 8 * hq * 512 floats.
hipError_t launch_prefill_mfma_probe(float* sink, int nq, int hq, hipStream_t s);
hipError_t launch_prefill_tile_levels(int32_t* out, int n_row_tiles, int n_kblocks, int q_offset,
                                      const LevelTable& lt, hipStream_t s);
hipError_t launch_decode(const DecodeArgs& a, hipStream_t s);
// The decode over the 8-bit cache (a.kv_exps).
hipError_t launch_decode_q8(const DecodeArgs& a, hipStream_t s);
// The merge of a call's split partials (nothing to do with one split in one workgroup).
hipError_t launch_decode_merge(const DecodeArgs& a, hipStream_t s);
// The decode over contiguous rows; every sequence has a.max_seq_len tokens.
hipError_t launch_decode_rows(const DecodeArgs& a, const DecodeRows& r, hipStream_t s);
// launch_decode with the workspace pointers taken from the device's fixed
// scratch (a.ws_ml and a.ws_o are set here).
hipError_t launch_decode_noalloc(DecodeArgs a, hipStream_t s);
// The streaming probe of the decode (measurement only): 8-wave workgroups
// over a.n_splits x a.hkv x a.batch; sink holds one word per wave.
hipError_t launch_decode_stream_probe(const DecodeArgs& a, uint32_t* sink, hipStream_t s);
hipError_t launch_decode_page_levels(int32_t* out, int n_pages, int seq_len, const LevelTable& lt,
                                     hipStream_t s);

}  // namespace atf
