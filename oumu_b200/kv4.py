"""The 4-bit paged KV cache of a set of layers: the buffers oumu_kv4_*, oumu_attn_decode_kv4* and oumu_pages_* work on
(include/oumu_attn.h) and the calls on them. Takes the place of the bf16 slots [slots][nk][maxlen][hd] of the reference
engine (src/model.rs:130-133) in 0.31 of their bytes, with memory for the positions takes hold instead of the longest
take's for every one, and the prompt held once for all takes that start from it (src/model.rs:705-717 copies it into
every slot)."""
import torch

from . import ops


class KV4Cache:
    """`layers` layers of `npages` pages for B takes of up to maxlen positions. `lens` (int32 [B], device) holds the takes'
    lengths; a caller that advances its own on the device (oumu_step_end_live) passes it. Everything but `missing` is
    enqueued on the current stream, without waiting for the GPU; calls to be captured take their takes as device tensors,
    not lists. With programmatic launches on (ops.set_pdl), `step` and `attend` may start while the kernel before them
    still runs: an ordinary launch (any of torch's) lies between free or compact and them (extend and fork end with one)."""

    def __init__(self, layers, B, nq, nk, hd, npages, maxlen, device="cuda", lens=None):
        self.layers, self.B, self.nq, self.nk, self.hd, self.npages = layers, B, nq, nk, hd, npages
        self.maxpages = -(-maxlen // ops.KV4_PAGE)
        if layers < 1 or B < 1 or npages < 1 or maxlen < 1:
            raise ValueError("a cache has layers, takes, pages and positions")
        if lens is not None and (lens.dtype is not torch.int32 or lens.numel() < B):
            raise ValueError("lens: int32 [B]")
        dev = torch.device(device)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
        self.pools = torch.empty((layers, npages, ops.kv4_page_bytes(nk, hd)), dtype=torch.uint8, device=dev)
        self.table = torch.full((B, self.maxpages), -1, dtype=torch.int32, device=dev)
        self.ref, self.lens = i32(npages), i32(B) if lens is None else lens
        # pages missing: [what extends lacked at most, what forks lacked in all] since `missing` was last asked, and of the
        # last call of each; [pages in use, pages moved]
        self.status, self._last, self.moved = i32(2), i32(2), i32(2)
        self.ws = ops.decode_kv4_workspace(B, nq, nk, hd, self.maxpages, dev)
        self._pages_ws = ops.pages_workspace(npages, dev)

    def _ids(self, takes):
        t = torch.as_tensor(takes, dtype=torch.int32)
        # from pinned memory: a copy from pageable memory waits for the stream
        return t if t.is_cuda else t.pin_memory().to(self.table.device, non_blocking=True)

    def extend(self, extra=0):
        """Pages for every take's first lens + extra positions. Those that the pool did not have are missing until
        `missing` is asked, whatever later calls find: what was to be written there is lost."""
        ops.pages_extend(self.table, self.ref, self.lens, extra, self._last[:1])
        torch.maximum(self.status[:1], self._last[:1], out=self.status[:1])

    def fork(self, src, dst):
        """Takes dst[i] continue where takes src[i] are, on shared pages (device int32 tensors, or lists). Takes for which
        no page was left end up empty; `missing` counts them."""
        ops.pages_fork(self.pools, self.table, self.ref, self.lens, self._ids(src), self._ids(dst), self._last[1:])
        self.status[1:].add_(self._last[1:])

    def missing(self):
        """Pages that extends (the most any one lacked) and forks (each) did not get since the last time this was asked;
        waits for the GPU."""
        n = sum(self.status.tolist())
        if n:
            self.status.zero_()
        return n

    def free(self, takes):
        ops.pages_free(self.table, self.ref, self.lens, self._ids(takes))

    def compact(self):
        """Pages in use to the front of the pools; moved = [pages in use, pages moved]."""
        ops.pages_compact(self.pools, self.table, self.ref, self._pages_ws, self.moved)

    def resize(self, npages):
        """`npages` pages from now on: those in use move to the front, into new pools, and the old pools' memory is free
        again. Waits for the GPU; graphs captured before hold the old pools and have to be captured anew."""
        self.compact()
        used = int(self.moved[0])
        if npages < max(used, 1):
            raise ValueError(f"{used} pages are in use")
        ws = ops.pages_workspace(npages, self.table.device)
        pools, ref = self.pools.new_empty((self.layers, npages, self.pools.shape[2])), self.ref.new_zeros(npages)
        pools[:, :used] = self.pools[:, :used]
        ref[:used] = self.ref[:used]
        torch.cuda.synchronize(self.table.device)  # other streams may still read the old pools
        self.pools, self.ref, self._pages_ws, self.npages = pools, ref, ws, npages

    def write(self, layer, qkv, rows, nq=None, start=None, count=None):
        """k and v of `rows` rows per take of qkv (nq q heads before them, by default the cache's) at start[s] + i."""
        ops.kv4_write(qkv, self.pools[layer], self.table, start, count, self.B, rows, self.nq if nq is None else nq,
                      self.nk, self.hd)

    def read(self, layer, kc, vc):
        """What the takes hold, as bf16 slots [B][nk][maxlen][hd]."""
        ops.kv4_read(self.pools[layer], self.table, self.lens, kc, vc, self.nk, self.hd)

    def attend(self, layer, qkv, out, scale=None):
        ops.attn_decode_kv4(qkv, self.pools[layer], out, self.ws, self.table, None, self.lens, self.B, self.nq, self.nk,
                            self.hd, self.hd ** -0.5 if scale is None else scale)

    def step(self, layer, qkv, out, cos_t=None, sin_t=None, scale=None, held=None):
        """One decode layer: rope, quantisation, cache write and attention of every take's newest position."""
        ops.attn_decode_kv4_step(qkv, self.pools[layer], out, self.ws, cos_t, sin_t, self.table, None, self.lens, self.B,
                                 self.nq, self.nk, self.hd, self.hd ** -0.5 if scale is None else scale, held=held)

    def nbytes(self):
        return self.pools.numel()
