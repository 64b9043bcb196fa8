"""Plain 64-bit forms of the operators on drafted tokens, written node by node from their definitions, and inputs for their tests."""
import math
import random

import torch


def chains(parents, n):
    """per node its ancestors, itself last"""
    out = []
    for i in range(n):
        p = parents[i]
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def attention(qkv, kc, vc, lens, parents, counts, Hq, starts=None, window=0):
    """-> (attention, sum of p |v|) [rows * nodes, Hq * D] in fp64, on the CPU"""
    qkv, kc, vc = qkv.detach().cpu().double(), kc.cpu(), vc.cpu()
    B, Hkv, _, D = kc.shape
    N = len(parents[0])
    out, size = (torch.zeros(B, N, Hq, D, dtype=torch.float64) for _ in range(2))
    x = qkv[:, :(Hq + 2 * Hkv) * D].reshape(B, N, Hq + 2 * Hkv, D)
    for b in range(B):
        fam = chains(parents[b], counts[b])
        for i, f in enumerate(fam):
            t = lens[b] + len(f) - 1
            lo = starts[b] if starts is not None else 0
            ctx = [j for j in range(lo, lens[b]) if not window or t - j < window]
            near = [j for j in f if not window or len(f) - len(fam[j]) < window]
            for h in range(Hq):
                g = h // (Hq // Hkv)
                k = torch.cat([kc[b, g, ctx].double(), x[b, near, Hq + g]])
                v = torch.cat([vc[b, g, ctx].double(), x[b, near, Hq + Hkv + g]])
                p = torch.softmax(k @ x[b, i, h] / math.sqrt(D), 0)
                out[b, i, h], size[b, i, h] = p @ v, p @ v.abs()
    return out.view(B * N, Hq * D), size.view(B * N, Hq * D)


def accept(parents, counts, tokens, choice):
    """-> per row (nodes of the path, the token after it)"""
    out = []
    for up, n, tok, ch in zip(parents, counts, tokens, choice):
        path = [0] if n else []
        while path:
            go = [i for i in range(n) if i and 0 <= up[i] < i and up[i] == path[-1] and tok[i] == ch[path[-1]]]
            if not go:
                break
            path.append(go[0])
        out.append((path, ch[path[-1]] if path else -1))
    return out


def alternatives(logits, targets, top, c):
    """fp64 on the CPU -> (logp, entropy, alternatives' logp, ids, E|z|, z of the targets, log S)"""
    l = logits.detach().cpu().double()
    T, V = l.shape
    raw = torch.where(torch.isnan(l), -math.inf, l)
    ids = torch.tensor([sorted(range(V), key=lambda j: (-r[j], j))[:top] for r in raw.tolist()]).view(T, top)
    z = (l - raw.amax(1, keepdim=True)) * c
    none = (l == -math.inf).all(1)
    ls = torch.logsumexp(z, 1)
    p = torch.exp(z - ls[:, None])
    ez = torch.where(p == 0, 0.0, p * z).sum(1)
    logp = torch.where(none[:, None], -math.inf, z - ls[:, None])
    ent = torch.where(none, 0.0, ls - ez)
    t = torch.full((T,), -1) if targets is None else targets.cpu().long()
    lp = torch.where(t >= 0, logp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    zt = torch.where(t >= 0, z.gather(1, t.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    return lp, ent, logp.gather(1, ids), ids, ez.abs(), zt.abs(), ls


def gradient(logits, targets, ids, c, g_lp, g_ent, g_top):
    """fp64 on the CPU: of sum g_lp logp + g_ent H + g_top alternatives -> (gradient, sum of its terms' sizes)"""
    l = logits.detach().cpu().double()
    z = (l - l.amax(1, keepdim=True)) * c
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    t, ids = targets.cpu().long(), ids.cpu()
    up = torch.zeros_like(p).scatter_add_(1, ids, g_top.cpu().double())
    gl = torch.where(t >= 0, g_lp.cpu().double(), 0.0)
    up.scatter_add_(1, t.clamp(min=0)[:, None], gl[:, None])
    total = up.sum(1, keepdim=True)
    ge = g_ent.cpu().double()[:, None]
    ent = -torch.where(p == 0, 0.0, p * logp).sum(1, keepdim=True)
    lh = torch.where(p == 0, 0.0, logp + ent)
    size = c * (up.abs() + p * (up.abs().sum(1, keepdim=True) + ge.abs() * (lh.abs() + ent + 1)))
    return c * (up - p * total - ge * p * lh), size


def trees(rows, nodes, seed, back=5):
    r = random.Random(seed)
    return [[-1] + [r.randint(max(0, i - back), i - 1) for i in range(1, nodes)] for _ in range(rows)]
