"""A batch of requests that share one prompt (or none): the pages of their own
rows in every layer, over the layers' compacted prompts.

The prompt's rows stay where they are, in a hot buffer of batch 1 per layer,
compacted or not, and are attended by all requests; a request's own rows live
in pages of one pool per layer.  Block tables, lengths and the free list are on
the device and are the same for all layers, so a step synchronises nothing and
can be captured: extend (once), attend (per layer), release (when tokens are
rejected or a request ends).
(No counterpart in the reference, whose caches are one dense tensor per layer
with one length for the whole batch, cache.py:145-148.)
"""

import torch

from . import ops


class SharedPromptBatch:
    def __init__(self, layers, requests, heads, head_dim, dtype, device, num_pages, page_size, max_rows):
        """heads: KV heads.  max_rows: the most own rows of one request.  All
        layers' pools together take layers * num_pages * page_size rows of
        2 * heads * head_dim elements."""
        if min(layers, requests, heads, num_pages, page_size, max_rows) < 1:
            raise ValueError("SharedPromptBatch: sizes must be at least 1")
        self.layers, self.requests, self.page_size = int(layers), int(requests), int(page_size)
        dev = torch.device(device)
        shape = (int(num_pages), int(heads), self.page_size, int(head_dim))
        # Rows are written before any read and stale ones are never attended,
        # so nothing is cleared.
        self.k_pages = [torch.empty(shape, dtype=dtype, device=dev) for _ in range(self.layers)]
        self.v_pages = [torch.empty(shape, dtype=dtype, device=dev) for _ in range(self.layers)]
        self.tables = torch.zeros((self.requests, -(-int(max_rows) // self.page_size)), dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.requests, dtype=torch.int32, device=dev)
        # taken from the end: page 0 first
        self.free_pages = torch.arange(int(num_pages) - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), int(num_pages), dtype=torch.int32, device=dev)
        self.prompts = [(None, None)] * self.layers
        self._step = None

    def set_prompt(self, layer, k, v=None):
        """The layer's shared prompt: a HotBuffer of batch 1, or k and v
        (1,H,S,D) or (H,S,D).  The rows are referred to, not copied: a buffer
        that is compacted or appended to afterwards is set again."""
        if v is None:
            if k.B != 1:
                raise ValueError(f"SharedPromptBatch: the prompt's buffer has batch {k.B}, not 1")
            k, v = k.keys, k.values
        self.prompts[layer] = (k, v)

    def extend(self, new_lens, num_tokens, max_new):
        """Begin a step: request b gets new_lens[b] (B,) int32 rows, max_new at
        most.  num_tokens: rows of the packed token batch, padding included.
        Returns the tokens' positions in their requests (-1: padding, or a
        request that does not fit and keeps its length); a prompt's length is
        the caller's to add."""
        self.lens, self.free_count, cu, slots, pos = ops.extend_pages(
            self.lens, new_lens, self.tables, self.free_pages, self.free_count, self.page_size, num_tokens,
            lens_out=self.lens, count_out=self.free_count)
        self._step = (cu, slots, max(1, int(max_new)))   # (a step of no tokens attends nothing)
        return pos

    def attend(self, layer, q, k, v, scaling, prefix_lens=None, out=None, return_lse=False):
        """One layer of the step: append the tokens' k, v (N,H,D) and attend
        their q (N,Hq,D) over the layer's prompt and their requests' own rows.
        prefix_lens (B,) int32: the prompt's rows that each request shares."""
        if self._step is None:
            raise RuntimeError("SharedPromptBatch: attend before extend")
        cu, slots, max_new = self._step
        kp, vp = self.prompts[layer]
        ops.append_paged(slots, k, v, self.k_pages[layer], self.v_pages[layer])
        return ops.prefix_attention(q, kp, vp, self.k_pages[layer], self.v_pages[layer], self.tables, self.lens,
                                    scaling, cu_new=cu, max_new=max_new, prefix_lens=prefix_lens, out=out,
                                    return_lse=return_lse)

    def release(self, keep_lens):
        """Keep each request's first keep_lens[b] (B,) int32 rows: 0 ends it,
        fewer than it has drop rejected tokens."""
        ops.release_pages(self.lens, keep_lens, self.tables, self.free_pages, self.free_count, self.page_size,
                          lens_out=self.lens, count_out=self.free_count)
        self._step = None   # (its tokens are no longer the requests' last)
