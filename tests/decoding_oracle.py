"""Plain restatements of the decoding operators (mmf_amd/decoding.py): loops over requests in Python, 64-bit floating point, on the CPU."""
import math

import torch


def plan(q_lens, kv_lens, tables, owned, free, top, page, rows, beams, shared):
    """Lists in, lists out; `tables`, `owned` and `free` (lists) are changed in place."""
    G, W, P = len(q_lens), beams, len(tables[0])
    up = lambda n: -(-n // page)
    for g in range(G):
        if q_lens[g] < 0:
            for w in range(W):
                for j in range(min(up(kv_lens[g]), P)):
                    if owned[g * W + w][j] >= 0:
                        free[top] = owned[g * W + w][j]
                        top += 1
    per = 1 if shared else W
    starts, granted, kv_out, copies, refused = [], [], [], [[-1] * 3 for _ in range(G * W)], 0
    slots, positions = [-1] * rows, [-1] * rows
    at, asked, left = 0, 0, top
    for g in range(G):
        q, kv, n = q_lens[g], kv_lens[g], max(q_lens[g], 0)
        starts += [at + w * n for w in range(per)]
        fits = kv + n <= P * page and at + per * n <= rows
        forks = [w for w in range(1, W) if not shared and n and fits and kv % page and owned[g * W + w][kv // page] < 0]
        need = per * (up(kv + n) - up(kv)) + len(forks) if n and fits else 0
        asked += need
        ok = q >= 0 and fits and (need == 0 or asked <= top)
        refused += q >= 0 and not ok
        granted.append(n if ok else 0)
        kv_out.append(0 if q < 0 else kv + granted[-1])
        if ok and n:
            for w in range(W):
                r = g * W + w
                for j in range(kv // page if w in forks else up(kv), up(kv + n)):
                    if shared and w:
                        tables[r][j], owned[r][j] = tables[g * W][j], -1
                        continue
                    left -= 1
                    if w in forks and j == kv // page:
                        copies[r] = [tables[r][j], free[left], kv % page]
                    tables[r][j] = owned[r][j] = free[left]
                for i in range(n if w < per else 0):
                    t = at + w * n + i
                    slots[t], positions[t] = tables[r][(kv + i) // page] * page + (kv + i) % page, kv + i
        at += per * n
    return starts, granted, kv_out, slots, positions, copies, left, refused


def attend(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, beams, causal, scale):
    """(out, bound): bound = sum_j p_j |v_j|, the scale of what a relative error of the probabilities does to the output; rows no request names are None in `named`."""
    q, kc, vc = q.double().cpu(), key_cache.double().cpu(), value_cache.double().cpu()
    tables, kv_lens, q_start, q_lens = tables.cpu(), kv_lens.tolist(), q_start.tolist(), q_lens.tolist()
    page, group = kc.shape[2], q.shape[1] // kc.shape[1]
    out, mag, reach = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], q.shape[1], dtype=torch.float64)
    named = torch.zeros(q.shape[0], dtype=torch.bool)
    for r, start in enumerate(q_start):
        n, m = kv_lens[r // beams], q_lens[r // beams]
        named[start:start + m] = True
        j = torch.arange(n)
        pages = tables[r].long()[j // page]
        k, v = kc[pages, :, j % page], vc[pages, :, j % page]              # [n, kv_heads, dim]
        for i in range(m):
            end = max(0, min(n, n - m + i + 1)) if causal else n
            if end == 0:
                continue
            for h in range(q.shape[1]):
                x = q[start + i, h]
                s = scale * (k[:end, h // group] @ x)
                p = torch.softmax(s, 0)
                out[start + i, h] = p @ v[:end, h // group]
                mag[start + i, h] = p @ v[:end, h // group].abs()
                reach[start + i, h] = (abs(scale) * (k[:end, h // group].abs() @ x.abs())).max() + (s.max() - s.min())
    return out, mag, reach, named


def select(logits, scores, finished, eos):
    """(scores, parents, tokens, finished, gap): gap = the smallest distance between unequal neighbours among the chosen and the first not chosen."""
    G, W = scores.shape
    V = logits.shape[1]
    out = []
    gap = math.inf
    for g in range(G):
        cand = torch.full((W, V), -math.inf, dtype=torch.float64)
        for w in range(W):
            x = logits[g * W + w].double().cpu()
            x = torch.where(torch.isnan(x), -math.inf, x)
            s = float(scores[g, w])
            s = -math.inf if s != s else s
            if bool(finished[g, w]):
                cand[w, eos] = s
            elif s > -math.inf and bool(torch.isfinite(x.max())):
                cand[w] = s + (x - torch.logsumexp(x, 0))
        v, i = torch.sort(cand.flatten(), descending=True, stable=True)
        d = (v[:W] - v[1:W + 1])[torch.isfinite(v[1:W + 1])] if W * V > W else (v[:-1] - v[1:])[torch.isfinite(v[1:])]
        d = d[d > 0]
        gap = min(gap, float(d.min()) if d.numel() else math.inf)
        out.append((v[:W], i[:W] // V, i[:W] % V))
    s, p, t = (torch.stack(x) for x in zip(*out))
    return s, p, t, finished.cpu().gather(1, p) | (t == eos), gap


def reorder(parents, kv_lens, tables, page):
    """(tables, copies) as lists."""
    G, W = len(parents), len(parents[0])
    new, copies = [], []
    for g in range(G):
        old = tables[g * W:(g + 1) * W]
        rows = [list(old[p]) for p in parents[g]]
        part = kv_lens[g] // page if kv_lens[g] % page else None
        idle = [w for w in range(W) if w not in parents[g]]
        seen = set()
        for w, p in enumerate(parents[g]):
            copy = [-1] * 3
            if part is not None and p in seen:
                src, dst = old[p][part], old[idle.pop(0)][part]
                rows[w][part] = dst
                copy = [src, dst, kv_lens[g] % page]
            seen.add(p)
            copies.append(copy)
        new += rows
    return new, copies
