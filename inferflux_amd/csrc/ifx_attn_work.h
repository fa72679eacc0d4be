// ifx_attn_work.h -- what a request comes to in the kernels of paged attention:
// row tiles or blocks of rows, and stages of keys.  Plain arithmetic on lengths,
// which the host runs as well (tests/cpp/test_attn_work.cpp).
//
// A request without new tokens comes to nothing, whatever it has in the cache: a
// slot of the batch that is idle, or every request of a plan that failed.  Its row
// numbers would otherwise start at -1.
#pragma once

#include "ifx_attn.h"

namespace ifx {

#define IFX_HOST_TOO __host__ __device__ __forceinline__

// Keys of a request that some rows of it see at most; more: of new tokens and of
// keys in front of them, up to where a stage begins.
IFX_HOST_TOO int window_keys(const AttnArgs &a, const Request &r, int64_t more) {
  const int64_t most = a.window + more;
  return a.window > 0 && most < r.kv ? static_cast<int>(most) : r.kv;
}
IFX_HOST_TOO int stages_of(int keys, int stage) {
  return keys > stage ? (keys + stage - 1) / stage : 1;
}
IFX_HOST_TOO int rows_keys(const AttnArgs &a, const Request &r) {
  return window_keys(a, r, static_cast<int64_t>(r.nq) + kRowKeys);
}

// {blocks of 32 rows, stages} in the kernels of few rows.  A request has no more
// than `most` blocks, those of max_q rows: the launch has workgroups for as many, and
// a request of more rows must not take the others'.
IFX_HOST_TOO int2 rows_units(const AttnArgs &a, const Request &r, int most) {
  const int blocks = (r.nq * a.G + kRowsMax - 1) / kRowsMax;
  return make_int2(blocks < most ? blocks : most, stages_of(rows_keys(a, r), kRowKeys));
}

// Whether a request goes as one block of rows among row tiles: it has no more rows
// than that, and no more keys than `most`.
IFX_HOST_TOO bool few_rows(const AttnArgs &a, const Request &r, int most) {
  return r.nq > 0 && r.nq * a.G <= kRowsMax && rows_keys(a, r) <= most;
}
// {row tiles, stages} in the 8-bit cache's kernel of many rows; of few rows {1,
// stages of few_keys}.  most: as few_rows', -1 where none goes that way.
IFX_HOST_TOO int2 tile_units_q8(const AttnArgs &a, const Request &r, int tile_rows, int few_keys, int most) {
  if (few_rows(a, r, most)) return make_int2(1, stages_of(rows_keys(a, r), few_keys));
  return make_int2((r.nq * a.G + tile_rows - 1) / tile_rows,
                   stages_of(window_keys(a, r, tile_rows + kTileKeys), kTileKeys));
}

// The workgroup's request, block of 32 of its rows and chunk of its keys.
struct RowsWork {
  Split split;
  int b, q0, nq, kv, R, ctx, lo0, block, z, ns, zbeg, zend;  // R: rows of the block
  bool tree;
};
// Chunks are of `unit` keys, a multiple of 32.  False: no such chunk, or no row.
IFX_HOST_TOO bool rows_work(const AttnArgs &a, const Split &split, int unit, int lds_rows, RowsWork &w) {
  w.split = split;
  if (w.split.chunk == 0) return false;
  w.b = w.split.b, w.q0 = w.split.req.q0, w.nq = w.split.req.nq, w.kv = w.split.req.kv;
  w.z = w.split.item / w.split.tiles, w.block = w.split.item - w.z * w.split.tiles;
  w.R = w.nq * a.G - kRowsMax * w.block;
  if (w.R <= 0) return false;
  if (w.R > lds_rows) w.R = lds_rows;
  w.ctx = w.kv - w.nq;  // position of the first row; below 0 it sees nothing
  w.tree = a.masks != nullptr;
  w.lo0 = a.window > 0 && w.ctx >= a.window ? w.ctx - a.window + 1 : 0;
  const int kbeg = w.lo0 & ~(kRowKeys - 1), kend = w.kv, chunk = w.split.chunk * unit;
  w.ns = kend > kbeg ? (kend - kbeg + chunk - 1) / chunk : 1;
  if (w.z >= w.ns) return false;
  w.zbeg = kbeg + w.z * chunk, w.zend = w.zbeg + chunk < kend ? w.zbeg + chunk : kend;
  return true;
}
// The row of the request that a lane takes as its block's n-th; those behind the
// last repeat it.
IFX_HOST_TOO int row_of_lane(const RowsWork &w, int n) { return kRowsMax * w.block + (n < w.R ? n : w.R - 1); }

}  // namespace ifx
