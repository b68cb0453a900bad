// wl_paged.h - KV caches in pages that sequences share: their layout, and the host interface of wl_paged.hip,
// wl_paged_attention.hip and wl_paged_select.hip.
//
// A pool is `pages` pages of `page` positions (a power of two, 16 to 256). Per page and KV head it holds page * HD halves of
// keys and as many of values, in the order in which the matrix cores take them, so that neither keys nor values are moved
// between lanes on the way (off: the position within its page):
//   keys    [off / 16][t][HD / 8][h][r][8] for off % 16 = 8 h + 4 t + r: eight values of a position are 16 bytes, and the
//           eight positions of one t lie side by side. Row 8 t + 4 h + r of a product's 16 keys is position 8 h + 4 t + r, so
//           the scores that a lane gets (rows 4 g .. 4 g + 3 of both halves of 32 keys) are eight positions in order;
//   values  [off / 8][HD][off % 8]: a channel's eight positions are 16 bytes, the operand that meets those scores.
// Bounds, where a pool keeps them: [pages][KH][2][HD] halves, the smallest and the largest key of each channel over the
// page's positions up to the last one stored (NaN where one of them is).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wl {

constexpr int kPgRows = 111;      // entries of a call that one launch takes, and one more: its arguments are 4 KB at most
constexpr int kPgUnit = 16;       // positions of a unit: a page holds whole ones
constexpr int kPgValues = 1 << 24;  // values of a row at most

struct PagePool {
  uint16_t *K = nullptr, *V = nullptr, *bounds = nullptr;
  const int32_t *table = nullptr;  // [sequences][width]
  int pages = 0, page = 0, shift = 0, KH = 0, HD = 0, width = 0;  // page = 1 << shift
  // halves before a KV head of a page
  __host__ __device__ int64_t at(int id, int kvh) const { return (((int64_t)id * KH + kvh) << shift) * HD; }
  // the page of a sequence's positions j * page ..; -1 where there is none
  __device__ int id(int seq, int j) const {
    const int i = table[(int64_t)seq * width + j];
    return (unsigned)i < (unsigned)pages ? i : -1;
  }
};

// Halves from a head's part of a page to value d of position off.
__host__ __device__ inline int pg_key(int off, int d, int HD) {
  return (off >> 4) * 16 * HD + (off >> 2 & 1) * 8 * HD + (d >> 3) * 64 + ((off >> 3 & 1) * 4 + (off & 3)) * 8 + (d & 7);
}
__host__ __device__ inline int pg_val(int off, int d, int HD) { return (off >> 3) * 8 * HD + d * 8 + (off & 7); }

// Entries of a call: rows row0[i] .. row0[i + 1] - 1 are positions pos[i].. of sequence seq[i].
struct PageRows {
  int n = 0;
  int seq[kPgRows], pos[kPgRows], row0[kPgRows + 1];
  __host__ __device__ int rows(int i) const { return row0[i + 1] - row0[i]; }
};

struct PageRope {
  int n, neox;  // rotated values of a head (0: none)
  double theta_scale, freq_scale;
  const float *freqs;
};

// base and scale as the other rotations take them
PageRope page_rope(int n, int neox, double base, double freq_scale, const float *freqs);

// q [rows][H * HD] rotated into qr (either may be null, with H 0), k [rows][KH * HD] rotated and v into the pages, and the
// bounds of the pages written to.
hipError_t paged_store_launch(const PagePool &p, const PageRows &r, const float *q, int H, const float *k, const float *v,
                              const PageRope &rope, float *qr, hipStream_t st);
// Positions pos0 .. pos0 + T - 1 of a sequence as rows k, v [T][KH * HD]; zeros where there is no page.
hipError_t paged_read_launch(const PagePool &p, int seq, int pos0, int T, float *k, float *v, hipStream_t st);

// Attention of the rows q [rows][H * HD]. prefix > 0: positions below it are the same pages for all entries, and may
// be read once for all rows. blocks [rows][KH][most] (or null): the pages that a row and KV head reads, in order, -1
// after the last.
int64_t paged_attention_scratch_floats(const PagePool &p, const PageRows &r, int H, int prefix, int most);
hipError_t paged_attention_launch(const PagePool &p, const PageRows &r, const float *q, int H, int prefix,
                                  const int32_t *blocks, int most, float scale, float *scratch, float *out, hipStream_t st);

// The pages each row and KV head takes: the first `first`, the last `recent`, and of the others the `top` whose score is
// largest: the largest, over the group's heads, of sum_d max(q_d lo_d, q_d hi_d), in 64 bits (a score that is not
// finite before all others; of equals the lower page).
struct PageSelect {
  int first, recent, top;
  __host__ __device__ int most() const { return first + recent + top; }
};
int64_t paged_select_scratch_bytes(const PagePool &p, const PageRows &r, const PageSelect &s);
hipError_t paged_select_launch(const PagePool &p, const PageRows &r, const float *q, int H, const PageSelect &s,
                               void *scratch, int32_t *blocks, hipStream_t st);

}  // namespace wl
