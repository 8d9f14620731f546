"""Plain models of the token pool and of tree attention over it (numpy, float64)."""
from __future__ import annotations

import numpy as np

POOL_EXHAUSTED, BAD_SLOT, BAD_COUNT = 1, 8, 16
MAX_TREE = 64


class TokenPoolModel:
    """The pool's page tables, free stack and lengths, request by request; with
    ``kv`` (any dtype, [pages, L, 2, H, page, dh]) its contents too."""

    def __init__(self, num_slots, max_tokens, num_pages, page_size, order=None, kv=None):
        self.page = page_size
        self.width = -(-max_tokens // page_size)
        self.table = np.full((num_slots, self.width), -1, np.int32)
        self.lengths = np.zeros(num_slots, np.int32)
        self.held = np.zeros(num_slots, np.int32)
        self.stack = list(range(num_pages) if order is None else order)
        self.error = 0
        self.kv = kv

    def begin_step(self, slots, counts, rows, parents=None):
        """The step's arrays; see parakeet_b200.tokens.TokenStep."""
        B = len(slots)
        start = np.zeros(B + 1, np.int64)
        start[1:] = np.cumsum(np.maximum(counts, 0))
        context = np.full(B, -1, np.int32)
        request = np.full(rows, -1, np.int32)
        position = np.zeros(rows, np.int32)
        slot_map = np.full(rows, -1, np.int32)
        masks = np.zeros(rows, np.uint64)
        seen, out_of_pages = set(), False
        for b, (s, n) in enumerate(zip(slots, counts)):
            r0, r1 = min(start[b], rows), min(start[b + 1], rows)
            request[r0:r1] = b
            if not 0 <= s < len(self.lengths) or s in seen:
                self.error |= BAD_SLOT
                continue
            seen.add(s)
            length = int(self.lengths[s])
            need = -(-(length + max(n, 0)) // self.page)
            if n < 0 or start[b + 1] > rows or (parents is not None and n > MAX_TREE) or \
                    need > self.width:
                self.error |= BAD_COUNT
                continue
            take = max(need - int(self.held[s]), 0)
            # the pages of a request that found too few are nobody's this step
            if take and (out_of_pages or take > len(self.stack)):
                self.error |= POOL_EXHAUSTED
                out_of_pages = True
                continue
            for i in range(take):
                self.table[s, self.held[s] + i] = self.stack.pop()
            self.held[s] += take
            context[b] = length
            depth = {}
            for j in range(n):
                r = r0 + j
                par = j - 1 if parents is None else int(parents[r])
                if par < -1 or par >= j:
                    self.error |= BAD_COUNT
                    par = -1
                depth[j] = depth[par] + 1 if par >= 0 else 0
                if parents is not None:
                    masks[r] = (masks[r0 + par] if par >= 0 else np.uint64(0)) | np.uint64(1 << j)
                position[r] = length + (depth[j] if parents is not None else j)
                tok = length + j
                slot_map[r] = self.table[s, tok // self.page] * self.page + tok % self.page
        return dict(row_start=np.minimum(start, rows).astype(np.int32), context=context,
                    row_request=request, positions=position, slot_map=slot_map,
                    masks=masks.view(np.int64) if parents is not None else None,
                    slots=list(slots), counts=list(counts))

    def append(self, layer, key, value, step):
        for r, at in enumerate(step["slot_map"]):
            if at >= 0:
                self.kv[at // self.page, layer, 0, :, at % self.page] = key[r]
                self.kv[at // self.page, layer, 1, :, at % self.page] = value[r]

    def end_step(self, step, last):
        for b, s in enumerate(step["slots"]):
            if step["context"][b] < 0:
                continue
            r0, n, keep = int(step["row_start"][b]), step["counts"][b], int(last[b])
            if not -1 <= keep < n:
                self.error |= BAD_COUNT
                keep = -1
            if step["masks"] is None:
                path = list(range(keep + 1))
            else:
                bits = int(step["masks"][r0 + keep]) & (2 ** 64 - 1) if keep >= 0 else 0
                path = [j for j in range(n) if bits >> j & 1]
            if self.kv is not None:
                at = [int(step["slot_map"][r0 + j]) for j in path]
                rows = [self.kv[a // self.page, :, :, :, a % self.page].copy() for a in at]
                for i, row in enumerate(rows):
                    a = int(step["slot_map"][r0 + i])
                    self.kv[a // self.page, :, :, :, a % self.page] = row
            self.lengths[s] = step["context"][b] + len(path)

    def truncate(self, slots, lengths):
        give, seen = [], set()
        for s, n in zip(slots, lengths):
            if not 0 <= s < len(self.lengths) or s in seen:
                self.error |= BAD_SLOT
                continue
            seen.add(s)
            if not 0 <= n <= self.lengths[s]:
                self.error |= BAD_COUNT
                continue
            keep = -(-int(n) // self.page)
            for i in range(keep, int(self.held[s])):
                give.append(self.table[s, i])
                self.table[s, i] = -1
            self.held[s] = min(keep, self.held[s])
            self.lengths[s] = n
        self.stack.extend(reversed(give))


def tree_attention(query, kv, layer, model, step, parents, scale):
    """float64 outputs [rows, H, dh] (NaN for rows of no or a refused request),
    and for error bounds: the weighted mean of |v|, and the largest sum of
    |q| |k| scale over the keys of each row."""
    q = np.asarray(query, np.float64)
    rows, H, dh = q.shape
    Hkv = kv.shape[3]
    out = np.full(q.shape, np.nan)
    mean_abs = np.zeros(q.shape)
    reach = np.zeros((rows, H))
    for b, s in enumerate(step["slots"]):
        ctx, r0, n = int(step["context"][b]), int(step["row_start"][b]), step["counts"][b]
        if ctx < 0:
            continue
        pages = model.table[s][: -(-(ctx + n) // model.page)]
        data = np.asarray(kv[pages, layer], np.float64)          # [pages, 2, Hkv, page, dh]
        key, value = (data[:, i].transpose(1, 0, 2, 3).reshape(Hkv, -1, dh)[:, : ctx + n]
                      for i in (0, 1))
        for j in range(n):
            own = {j}
            if parents is None:
                own.update(range(j))
            else:
                at = j
                while True:
                    at = int(parents[r0 + at])
                    if not 0 <= at < max(own):
                        break
                    own.add(at)
            see = list(range(ctx)) + [ctx + i for i in sorted(own)]
            for h in range(H):
                k, v = key[h // (H // Hkv)][see], value[h // (H // Hkv)][see]
                t = k @ q[r0 + j, h] * scale
                p = np.exp(t - t.max())
                p /= p.sum()
                out[r0 + j, h] = p @ v
                mean_abs[r0 + j, h] = p @ np.abs(v)
                reach[r0 + j, h] = (np.abs(k) @ np.abs(q[r0 + j, h])).max() * scale
    return out, mean_abs, reach
