"""The 8-bit paged KV cache: pages of e4m3 codes with a power of two per page and KV
head, the block tables and slots of a step made on the device, attention over
whole contexts and over selected pages. Addresses are device addresses; calls are queued on the
device handle's stream and return without waiting."""
from __future__ import annotations

from operator import index

from ._lib import call, lib
from .device import Device

PAGE = 16  # positions of a page


def page_bytes(kv_heads: int, head_dim: int) -> int:
    """Bytes of a page (0 for head sizes that the pool does not take)."""
    return int(lib().pgd_kv8_page_bytes(kv_heads, head_dim))


def kv_tables_dev(dev: Device, block: int, nseq: int, lens_ptr: int, counts_ptr: int, tables_ptr: int, max_blocks: int,
                  free_ptr: int, n_free: int, taken_ptr: int, rows: int, new_lens_ptr: int, new_taken_ptr: int,
                  row_start_ptr: int, seq_of_row_ptr: int, pos_of_row_ptr: int, slots_ptr: int, status_ptr: int) -> None:
    """A step's pages, row starts, sequences, positions and slots from its lengths and row counts."""
    call("pgd_kv_tables_dev", dev.handle, block, nseq, index(lens_ptr or 0), index(counts_ptr or 0),
         index(tables_ptr or 0), max_blocks, index(free_ptr or 0), n_free, index(taken_ptr or 0), rows,
         index(new_lens_ptr or 0), index(new_taken_ptr or 0), index(row_start_ptr or 0), index(seq_of_row_ptr or 0),
         index(pos_of_row_ptr or 0), index(slots_ptr or 0), index(status_ptr or 0))


class Kv8Pool:
    """n_pages pages for kv_heads heads of head_dim (64, 128 or 256): in device memory of its own, or at ptr."""

    def __init__(self, dev: Device, kv_heads: int, head_dim: int, n_pages: int, ptr: int = 0):
        self.dev, self.kv_heads, self.head_dim, self.n_pages = dev, kv_heads, head_dim, n_pages
        self.owned = 0
        size = page_bytes(kv_heads, head_dim)
        if not size or n_pages < 1:
            raise ValueError(f"no pages for kv_heads {kv_heads}, head_dim {head_dim}, n_pages {n_pages}")
        self.page_bytes = size
        if not ptr:
            ptr = self.owned = dev.alloc(size * n_pages)
        self.ptr = index(ptr)

    def free(self) -> None:
        if self.owned and self.dev.handle:
            self.dev.free(self.owned)
        self.owned = self.ptr = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def _pool(self):
        return self.dev.handle, self.ptr, self.n_pages, self.kv_heads, self.head_dim

    def append_dev(self, k_ptr: int, ldk: int, v_ptr: int, ldv: int, x_type: int, slots_ptr: int, rows: int) -> None:
        """Rows of K and V (f32 / f16 / bf16) into their slots."""
        call("pgd_kv8_append_dev", *self._pool(), index(k_ptr or 0), ldk, index(v_ptr or 0), ldv, x_type,
             index(slots_ptr or 0), rows)

    def read_dev(self, slots_ptr: int, rows: int, k_ptr: int, ldk: int, v_ptr: int, ldv: int) -> None:
        """The f32 values of the positions at the slots."""
        call("pgd_kv8_read_dev", *self._pool(), index(slots_ptr or 0), rows, index(k_ptr or 0), ldk, index(v_ptr or 0),
             ldv)

    def attn_ws_bytes(self, heads: int, nseq: int, max_blocks: int, rows: int, max_rows: int | None = None) -> int:
        """Workspace of attn_dev for calls of up to these numbers (max_rows None: whatever the call will say)."""
        return int(lib().pgd_attn_kv8_rows_ws_bytes(heads, self.kv_heads, self.head_dim, nseq, max_blocks, rows,
                                                    max(rows, 0) if max_rows is None else max_rows))

    def attn_dev(self, heads: int, q_ptr: int, ldq: int, x_type: int, nseq: int, row_start_ptr: int, lens_ptr: int,
                 tables_ptr: int, max_blocks: int, rows: int, max_rows: int, out_ptr: int, ldo: int, ws_ptr: int,
                 ws_bytes: int, gate_ptr: int = 0, ldg: int = 0) -> None:
        """Causal attention of each sequence's latest rows over its context."""
        call("pgd_attn_kv8_dev", *self._pool(), heads, index(q_ptr or 0), ldq, x_type, nseq, index(row_start_ptr or 0),
             index(lens_ptr or 0), index(tables_ptr or 0), max_blocks, rows, max_rows, index(out_ptr or 0), ldo,
             index(gate_ptr or 0), ldg, index(ws_ptr or 0), ws_bytes)

    def sparse_ws_bytes(self, heads: int, rows: int, max_blocks: int, top: int) -> int:
        """Workspace of select_dev and attn_sparse_dev, one after the other."""
        return int(lib().pgd_kv8_sparse_ws_bytes(heads, self.kv_heads, self.head_dim, rows, max_blocks, top))

    def select_dev(self, heads: int, q_ptr: int, ldq: int, x_type: int, nseq: int, row_start_ptr: int, lens_ptr: int,
                   tables_ptr: int, max_blocks: int, rows: int, top: int, sinks: int, recent: int, sel_ptr: int,
                   count_ptr: int, ws_ptr: int, ws_bytes: int) -> None:
        """Per (row, KV head) the pages of the highest bounds on q.k, the first `sinks` and last `recent` among them."""
        call("pgd_kv8_select_dev", *self._pool(), heads, index(q_ptr or 0), ldq, x_type, nseq,
             index(row_start_ptr or 0), index(lens_ptr or 0), index(tables_ptr or 0), max_blocks, rows, top, sinks,
             recent, index(sel_ptr or 0), index(count_ptr or 0), index(ws_ptr or 0), ws_bytes)

    def attn_sparse_dev(self, heads: int, q_ptr: int, ldq: int, x_type: int, nseq: int, row_start_ptr: int,
                        lens_ptr: int, tables_ptr: int, max_blocks: int, rows: int, top: int, sel_ptr: int,
                        count_ptr: int, out_ptr: int, ldo: int, ws_ptr: int, ws_bytes: int, gate_ptr: int = 0,
                        ldg: int = 0) -> None:
        """attn_dev over the selected pages alone."""
        call("pgd_attn_kv8_sparse_dev", *self._pool(), heads, index(q_ptr or 0), ldq, x_type, nseq,
             index(row_start_ptr or 0), index(lens_ptr or 0), index(tables_ptr or 0), max_blocks, rows, top,
             index(sel_ptr or 0), index(count_ptr or 0), index(out_ptr or 0), ldo, index(gate_ptr or 0), ldg,
             index(ws_ptr or 0), ws_bytes)
