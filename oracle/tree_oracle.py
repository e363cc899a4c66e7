"""Plain restatement of the operators of a step with drafted trees: tables from request lengths, the walk, the moves in whole
numbers and Python lists, attention in 64 bits."""
from __future__ import annotations

import torch


class BlockState:
    """The allocator as lists: tables[r] (columns, -1 where there is none), owned[r], a stack of free ids."""

    def __init__(self, tables, owned, free, block_size):
        self.tables = [list(r) for r in tables]
        self.owned, self.free, self.block_size = list(owned), list(free), block_size
        self.left_out = 0

    def step(self, rows, cached, new, num_tokens, parents=None, words=0, buffer_rows=None):
        bs, cols, n = self.block_size, len(self.tables[0]), len(cached)
        rows = list(range(n)) if rows is None else list(rows)
        free_before, upto, at = len(self.free), 0, 0
        taken = []                                      # (row, ids) in the order of the batch
        cu_q, cu_k, ctx, bt = [0], [0], [], []
        slots, positions = [-1] * num_tokens, [0] * num_tokens
        masks = [[0] * words for _ in range(num_tokens)]
        self.left_out = 0
        for i in range(n):
            c, k = max(cached[i], 0), max(new[i], 0)
            ok = 0 <= rows[i] < len(self.tables) and rows[i] not in rows[:i]
            need = -(-(c + k) // bs)
            held = max(0, min(self.owned[rows[i]], cols)) if ok else 0
            ok = ok and need <= cols and not (parents is not None and k > 64 * words) and at + k <= num_tokens
            want = max(need - held, 0) if ok else 0
            upto += want
            ok = ok and (want == 0 or upto <= free_before)
            row = [-1] * cols
            if ok:
                mine = self.tables[rows[i]]
                for j in range(want):
                    mine[held + j] = self.free[free_before - 1 - (upto - want + j)]
                if want:
                    self.owned[rows[i]] = need
                    taken.append(want)
                row[:need] = mine[:need]
                for j in range(k):
                    p = c + j
                    slots[at + j] = row[p // bs] * bs + p % bs
                    positions[at + j] = p
                    if parents is not None:
                        node, depth = j, 0
                        while True:
                            masks[at + j][node // 64] |= 1 << (node % 64)
                            up = parents[at + node]
                            if not 0 <= up < node:
                                break
                            node, depth = up, depth + 1
                        positions[at + j] = c + depth
            else:
                self.left_out += 1
            at += k
            cu_q.append(min(at, num_tokens))
            ctx.append(c + k if ok else 0)
            cu_k.append(cu_k[-1] + ctx[-1])
            bt.append(row)
        if sum(taken):
            del self.free[-sum(taken):]
        extra = (buffer_rows or n) - n
        as_signed = [[w - (1 << 64) if w >> 63 else w for w in m] for m in masks]
        return dict(cu_q=cu_q + cu_q[-1:] * extra, cu_k=cu_k + cu_k[-1:] * extra, ctx=ctx + [0] * extra, slots=slots,
                    positions=positions, tables=bt, masks=as_signed)

    def release(self, rows, keep):
        back = []
        rows = list(range(len(keep))) if rows is None else list(rows)
        for i, r in enumerate(rows):
            if not 0 <= r < len(self.tables) or r in rows[:i]:
                continue
            k = min(-(-max(keep[i], 0) // self.block_size), self.owned[r])
            back += self.tables[r][k:self.owned[r]]
            self.tables[r][k:self.owned[r]] = [-1] * (self.owned[r] - k)
            self.owned[r] = k
        self.free += back[::-1]


def accept_tree_ref(draft, target, parents, cu, cached, ctx, max_path):
    accepted, paths, tokens, lens = [], [], [], []
    for i in range(len(cached)):
        lo, n = cu[i], cu[i + 1] - cu[i]
        path = []
        if ctx[i] > 0 and n > 0:
            path = [0]
            while len(path) < max_path:
                cur = path[-1]
                after = [c for c in range(cur + 1, n) if parents[lo + c] == cur and draft[lo + c] == target[lo + cur]]
                if not after:
                    break
                path.append(after[0])
        pad = [-1] * (max_path - len(path))
        accepted.append(len(path))
        paths.append(path + pad)
        tokens.append([target[lo + c] for c in path] + pad)
        lens.append(cached[i] + len(path))
    return accepted, paths, tokens, lens


def compact_ref(cache, path, accepted, start, tables, block_size):
    """cache (planes, blocks, block size, ...) on the CPU, changed in place: all rows are read before any is written."""
    before = cache.clone()
    for i, p in enumerate(path):
        for k in range(min(accepted[i], len(p))):
            if p[k] <= k:
                continue
            a, b = start[i] + p[k], start[i] + k
            ca, cb = a // block_size, b // block_size
            if b < 0 or max(ca, cb) >= len(tables[i]):
                continue
            ta, tb = tables[i][ca], tables[i][cb]
            if 0 <= ta < cache.shape[1] and 0 <= tb < cache.shape[1]:
                cache[:, tb, b % block_size] = before[:, ta, a % block_size]


def tree_attn_ref(q, k_cache, v_cache, cu, ctx, tables, masks, scale):
    """(out, weight): attention in 64 bits, and the same with |v|, the size that roundings of the probabilities act on.
    Rows outside cu are zero.  masks: (tokens, words) int64 or None."""
    total, H, D = q.shape
    bs, hkv = k_cache.shape[1], k_cache.shape[2]
    G = H // hkv
    out, weight = torch.zeros(total, H, D, dtype=torch.float64), torch.zeros(total, H, D, dtype=torch.float64)
    for i in range(len(ctx)):
        lo, hi, n = cu[i], cu[i + 1], max(ctx[i], 0)
        if hi <= lo or n == 0:
            continue
        pos = torch.arange(n)
        block = torch.tensor(tables[i])[pos // bs]
        k, v = k_cache[block, pos % bs].double(), v_cache[block, pos % bs].double()
        node = pos - (n - (hi - lo))                                                 # (keys)
        for j in range(hi - lo):
            if masks is None:
                sees = node <= j
            else:
                words = masks[lo + j].tolist()
                bit = [(words[x // 64] >> (x % 64)) & 1 if 0 <= x < 64 * len(words) else 0 for x in node.tolist()[max(0, n - (hi - lo)):]]
                sees = node < 0
                sees[max(0, n - (hi - lo)):] = torch.tensor(bit, dtype=torch.bool)
            if not sees.any():
                continue
            s = torch.einsum("hgd,shd->hgs", q[lo + j].double().view(hkv, G, D), k) * scale
            p = torch.softmax(s.masked_fill(~sees, float("-inf")), -1)
            out[lo + j] = torch.einsum("hgs,shd->hgd", p, v).reshape(H, D)
            weight[lo + j] = torch.einsum("hgs,shd->hgd", p, v.abs()).reshape(H, D)
    return out, weight
