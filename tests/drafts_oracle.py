"""The drafted step's operators in 64 bits on the CPU, one value after another, and the bounds that the
GPU results are held to.

Rounding of a type is off by at most u = eps / 2 of the value.  An attention level, per output:

* a score is a product of d terms summed in fp32 (d + 2 roundings of 2^-24 of sum |q k|), scaled,
  clamped and shifted by a bias (4 more of its size), then exp2 in fp32 (2^-22 relative): relative
  error of a weight and of their sum at most r = 2 (largest score error) + 2^-21;
* the weights of cached positions enter the second product rounded to the type (16-bit types): u;
  a middle level's cached values v * msg are rounded too: u;
* the sum itself: (n + 64) 2^-24 for n terms in fp32;
* the deeper level's error enters through the drafted values (linearly) and logsumexps (r);
* the stored result is rounded once: u of the output, and below the smallest normal number tiny, where
  the type's steps stop shrinking, u tiny (float16: steps of 2^-24 below 2^-14, so half a step is 2^-25
  whatever the value, while u |y| goes to 0 with y).
"""

import math

import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def stored(y, dtype):
    """Half a step of the type at y."""
    return unit(dtype) * y.abs().clamp(min=torch.finfo(dtype).tiny)


def walk_tree(parents):
    """[ancestors and itself] per node, None for an absent one, of one row's parents."""
    out = []
    for t, p in enumerate(parents):
        if p == -1:
            out.append([t])
        elif 0 <= p < t and out[p] is not None:
            out.append(out[p] + [t])
        else:
            out.append(None)
    return out


def attend(q1, cache, lens, parents, scale, softclamp):
    """(out, msgs, lses) and their bounds, from CPU copies of a DraftCache's buffers (a dict)."""
    B, H, T, d = q1.shape
    hk, order = cache["qs"][0].shape[1], len(cache["qs"])
    dt = q1.dtype
    u = unit(dt)
    up = u if dt != torch.float32 else 0.0
    D = lambda x: x.double()  # noqa: E731
    res = [torch.zeros(B, H, T, d, dtype=torch.float64)]
    res += [torch.zeros(B, hk, T, d, dtype=torch.float64) for _ in range(order - 1)]
    res += [torch.zeros(B, hk, T, dtype=torch.float64) for _ in range(order - 1)]
    tol = [torch.zeros_like(x) for x in res]
    for b in range(B):
        n = lens[b]
        tree = walk_tree(parents[b])
        for kv in range(hk):
            msg = emsg = lse = else_ = None
            for t in range(order):
                lvl = order - 1 - t
                heads = range(kv * (H // hk), (kv + 1) * (H // hk)) if lvl == 0 else [kv]
                nmsg = torch.zeros(T, d, dtype=torch.float64)
                nem, nl, nel = torch.zeros_like(nmsg), torch.zeros(T).double(), torch.zeros(T).double()
                for h in heads:
                    for i in range(T):
                        if tree[i] is None:
                            continue
                        s = tree[i]
                        q = D(q1[b, h, i] if lvl == 0 else cache["draft_qs"][lvl - 1][b, h, i])
                        k = torch.cat([D(cache["qs"][lvl][b, kv, :n]), D(cache["draft_qs"][lvl][b, kv, s])])
                        x = (k @ q) * scale
                        ex = (d + 6) * F32 * abs(scale) * (k.abs() @ q.abs())
                        if softclamp:
                            x = softclamp * torch.tanh(x / softclamp)
                            ex = ex + 8 * F32 * softclamp
                        eb = 0.0
                        if t:
                            bias = torch.cat([D(cache["lses"][t - 1][b, kv, :n]), lse[s]])
                            eb = torch.cat([torch.zeros(n).double(), else_[s]])
                            x = x + bias
                            ex = ex + 6 * F32 * bias.abs()
                        if t == 0:
                            v = torch.cat([D(cache["vs"][-1][b, kv, :n]), D(cache["draft_vs"][-1][b, kv, s])])
                            ev = torch.zeros_like(v)
                        else:
                            v = torch.cat([D(cache["msgs"][t - 1][b, kv, :n]), msg[s]])
                            ev = torch.cat([torch.zeros(n, d).double(), emsg[s]])
                            if lvl:
                                w = torch.cat([D(cache["vs"][lvl - 1][b, kv, :n]),
                                               D(cache["draft_vs"][lvl - 1][b, kv, s])])
                                v, ev = v * w, ev * w.abs()
                                ev[:n] += u * v[:n].abs()
                                ev[n:] += 2 * F32 * v[n:].abs()
                        x = torch.where(x.isnan(), -math.inf, x)
                        z = torch.logsumexp(x, 0)
                        p = torch.exp(x - z)
                        live = p > 0
                        r = 2 * ((ex + eb + 4 * F32 * x.abs()) * live).nan_to_num(0, 0, 0).max() + 2.0 ** -21
                        p, v, ev = p[live], v[live], ev[live]
                        o = p @ v
                        rel = torch.full((len(p),), float(r) + (n + T + 64) * F32).double()
                        rel[live.nonzero()[:, 0] < n] += up
                        e = (p * rel) @ v.abs() + p @ ev
                        if lvl == 0:
                            res[0][b, h, i], tol[0][b, h, i] = o, e + stored(o, dt)
                        else:
                            nmsg[i], nem[i] = o, e
                            nl[i], nel[i] = z, r + (n + T + 64) * F32 + 4 * F32 * abs(z)
                if lvl:
                    msg, emsg, lse, else_ = nmsg, nem, nl, nel
                    res[1 + t][b, kv], tol[1 + t][b, kv] = msg, emsg + stored(msg, dt)
                    res[order + t][b, kv], tol[order + t][b, kv] = lse, else_
    return res, tol


def rows(src, weight, eps, angles):
    """The norm (weight not None) and rotation (angles [B, T, r] or None) of [B, h, T, d], and the bound."""
    x = src.double()
    d = x.shape[-1]
    y, e = x, torch.zeros_like(x)
    if weight is not None:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
        e = (d / 2 + 8) * F32 * y.abs()
    if angles is not None:
        a = angles.double()[:, None]
        r = a.shape[-1]
        z, ez = y.clone(), e.clone()
        c, s = a.cos(), a.sin()
        z[..., 0:r:2] = y[..., 0:r:2] * c[..., 0::2] - y[..., 1:r:2] * s[..., 0::2]
        z[..., 1:r:2] = y[..., 1:r:2] * c[..., 1::2] + y[..., 0:r:2] * s[..., 1::2]
        both = y[..., 0:r:2].abs() + y[..., 1:r:2].abs()
        eboth = e[..., 0:r:2] + e[..., 1:r:2] + 6 * F32 * both
        ez[..., 0:r:2] = eboth
        ez[..., 1:r:2] = eboth
        y, e = z, ez
    if weight is None and angles is None:
        return y, e
    return y, e + stored(y, src.dtype)


def verify(logits, tokens, parents, uniforms, noise, temperature, probs):
    """Per row: (path, token), and the smallest relative distance of a decision from its border."""
    B, T, V = logits.shape
    out, margin = [], math.inf
    for b in range(B):
        tree = walk_tree(parents[b])
        temp = 0.0 if uniforms is None else 1.0 if temperature is None else float(temperature[b])

        def target(t):
            x = logits[b, t].double()
            if temp > 0:
                return torch.softmax(x / temp, 0)
            p = torch.zeros(V, dtype=torch.float64)
            p[(x == x.max()).nonzero()[0, 0]] = 1.0
            return p

        if tree[0] is None:
            out.append(([], -1))
            continue
        cur, path, p = 0, [0], target(0)
        for t in range(1, T):
            if tree[t] is None or parents[b][t] != cur:
                continue
            x = int(tokens[b, t])
            inside = 0 <= x < V
            px = float(p[x]) if inside else 0.0
            q = probs[b, cur].double() if probs is not None else None
            qx = 1.0 if q is None or not inside else float(q[x])
            uq = (float(uniforms[b, t]) if temp > 0 else 0.0) * qx
            if temp > 0 and px > 0:
                margin = min(margin, abs(uq - px) / px)
            if uq < px:
                cur, p = t, target(t)
                path.append(t)
                continue
            rest = p.clone()
            if q is not None:
                rest = (p - q).clamp(min=0)
            elif inside:
                rest[x] = 0
            if rest.sum() > 0:
                p = rest / rest.sum()
        if temp > 0:
            key = torch.where(p > 0, p / noise[b].double(), -1.0)
            top = key.sort(descending=True).values
            margin = min(margin, float((top[0] - top[1]) / top[0])) if V > 1 else margin
            out.append((path, int((key == key.max()).nonzero()[0, 0])))
        else:
            out.append((path, int(p.argmax())))
    return out, margin
