"""Plain definitions of the block-attention operators in 64 bits, with a bound of what rounding may do to them.

Test infrastructure (like the rest of oracle/): dense, one head of one sequence at a time, nothing shared with the package.  `u` is
half a step of a type relative to the value: float32 2^-24, bfloat16 2^-8."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def norm_rotate(x, w, turns, positions, eps=1e-6):
    """x (B, L, H, D) -> float64"""
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if turns is not None and turns.numel():
        h = turns.numel()
        ang = positions.double()[..., None] * turns.double()
        ang = 2 * math.pi * (ang - ang.floor())
        z = torch.complex(y[..., :h].contiguous(), y[..., h:2 * h].contiguous()) * torch.polar(torch.ones_like(ang), ang)[:, :, None]
        y = torch.cat([z.real, z.imag, y[..., 2 * h:]], -1)
    return y


def summary(k, block, klen):
    B, Lk, Hk, D = k.shape
    out = torch.zeros(B, -(-Lk // block), Hk, D, dtype=torch.float64)
    for b in range(B):
        n = Lk if klen is None else int(klen[b])
        for j in range(-(-n // block)):
            out[b, j] = k[b, j * block:min(n, (j + 1) * block)].double().mean(0)
    return out


def select(q, summ, n, block, qb, Lk, causal, qlen, klen, sink=1, local=1):
    B, Lq, Hq, D = q.shape
    nb, Hk = summ.shape[1:3]
    G, ng = Hq // Hk, -(-Lq // qb)
    sel = torch.full((B, Hk, ng, n), -1, dtype=torch.int32)
    for b in range(B):
        ql = Lq if qlen is None else int(qlen[b])
        kl = Lk if klen is None else int(klen[b])
        for g in range(ng):
            rows = range(g * qb, min((g + 1) * qb, ql))
            if not len(rows):
                continue
            last = kl - ql + rows[-1]
            for h in range(Hk):
                x = q[b, rows[0]:rows[-1] + 1, h * G:(h + 1) * G].double().sum((0, 1))
                score = (summ[b, :, h].double() @ x).tolist()
                may = [j for j in range(nb) if j * block < kl and (not causal or j * block <= last)]

                def rank(j):
                    must = j < sink or abs(j - last // block) < local
                    s = math.inf if must else score[j]
                    return (0 if must else 1, 1 if s != s else 0, -s if s == s else 0.0, j)
                best = sorted(sorted(may, key=rank)[:n])
                sel[b, h, g, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return sel


def visible(sel_row, block, Lk, klen, causal, qkey):
    """keys that one query sees: bool (Lk,)"""
    m = torch.zeros(Lk, dtype=torch.bool)
    top = -1
    for e in sel_row.tolist():
        if e < 0 or e * block >= Lk or e <= top:
            continue
        top = e
        m[e * block:(e + 1) * block] = True
    m[max(0, klen):] = False
    if causal:
        m[max(0, qkey + 1):] = False
    return m


def weigh(P, V, mask):
    """P V over the visible keys only: what a masked key holds does not matter"""
    if torch.isfinite(V).all():
        return P @ V
    return torch.stack([P[i, m] @ V[m] for i, m in enumerate(mask)])


def attention(q, k, v, sel, block, qb, scale, causal, qlen, klen, bucket_of=None, bias=None, q_pos=None, k_pos=None, dout=None,
              parts=1):
    """float64 results and element-wise bounds of the error of a computation whose products and sums are fp32 and whose probabilities
    and score gradients are held in `parts` numbers of the inputs' type in front of the second products (each rounds what the ones
    before it left over):
    {name: (value, bound)} of out, lse, and with dout dq, dk, dv, dbias."""
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1:3]
    G, u = Hq // Hk, U[q.dtype]
    up = u ** parts if q.dtype != torch.float32 else 0.0
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    names = {'out': z(*q.shape), 'lse': torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64)}
    if dout is not None:
        names.update(dq=z(*q.shape), dk=z(*k.shape), dv=z(*k.shape))
        if bias is not None:
            names['dbias'] = z(*bias.shape)
    val, err = {n: t.clone() for n, t in names.items()}, {n: torch.zeros_like(t) for n, t in names.items()}
    for b in range(B):
        ql = Lq if qlen is None else int(qlen[b])
        kl = Lk if klen is None else int(klen[b])
        if ql == 0:
            continue
        for h in range(Hq):
            c = h // G
            K, V = k[b, :, c].double().clone(), v[b, :, c].double().clone()
            K[kl:], V[kl:] = 0, 0
            Q = q[b, :ql, h].double()
            mask = torch.stack([visible(sel[b, c, i // qb], block, Lk, kl, causal, kl - ql + i) for i in range(ql)])
            S = Q @ K.T * scale
            # fp32: D products and sums, the scaling, the bias, then (S - max) * log2(e) and the exponential's own step
            eS = (D + 2) * U32 * abs(scale) * (Q.abs() @ K.abs().T)
            if bias is not None:
                qp = torch.arange(ql) + kl - ql if q_pos is None else q_pos[b, :ql].long()
                kp = torch.arange(Lk) if k_pos is None else k_pos[b].long()
                md = bucket_of.numel() // 2
                bucket = bucket_of.long()[(kp[None] - qp[:, None]).clamp(-md, md) + md]
                mask &= bias[:, h][bucket] >= -1e30                             # (lower ones mask)
                S = S + bias[:, h].double()[bucket]
                eS = eS + 2 * U32 * S.abs()
            S = S.masked_fill(~mask, -math.inf)
            some = mask.any(1)
            top = S.amax(1, keepdim=True).masked_fill(~some[:, None], 0.0)
            P = (S - top).exp().masked_fill(~mask, 0.0)
            L = P.sum(1, keepdim=True).masked_fill(~some[:, None], 1.0)
            P = P / L
            eS = eS.masked_fill(~mask, 0.0) + 4 * U32 * (S - top).abs().masked_fill(~mask, 0.0)
            worst = eS.amax(1, keepdim=True)
            n = mask.sum(1, keepdim=True)
            eP = 2 * worst + (n + 16) * U32                                    # relative, of a probability (its sum included)
            O, A = weigh(P, V, mask), weigh(P, V.abs(), mask)
            val['out'][b, :ql, h] = O
            err['out'][b, :ql, h] = A * (up + eP + (n + 16) * U32) + u * O.abs()
            val['lse'][b, h, :ql] = torch.where(some, top[:, 0] + L[:, 0].log(), torch.tensor(-math.inf, dtype=torch.float64))
            err['lse'][b, h, :ql] = (eP[:, 0] + 16 * U32 * (1 + top[:, 0].abs() + L[:, 0].log().abs()))
            if dout is None:
                continue
            g = dout[b, :ql, h].double()
            dP = g @ V.T
            delta = (g * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            eO = A * (eP + (n + 16) * U32) + 2 * U32 * O.abs()                 # the saved result is not rounded to the type
            e_in = (D + 2) * U32 * (g.abs() @ V.abs().T) + (g.abs() * eO).sum(1, keepdim=True) + (D + 2) * U32 * (g.abs() * O.abs()).sum(1, keepdim=True)
            el = (err['lse'][b, h, :ql] + 4 * U32 * val['lse'][b, h, :ql].abs().masked_fill(~some, 0.0))[:, None]
            eQ = eP + el + 4 * U32 * S.abs().masked_fill(~mask, 0.0)           # P again, from lse
            eD = P * e_in + (eQ + 4 * U32) * dS.abs()
            eT = eD + up * dS.abs()      # rounded in front of the product
            rows = ql + 16
            val['dq'][b, :ql, h] = dS @ K * scale
            err['dq'][b, :ql, h] = abs(scale) * ((eT + (n + 16) * U32 * dS.abs()) @ K.abs()) + u * (dS @ K * scale).abs()
            val['dk'][b, :, c] += dS.T @ Q * scale
            err['dk'][b, :, c] += abs(scale) * ((eT + G * rows * U32 * dS.abs()).T @ Q.abs())
            val['dv'][b, :, c] += P.T @ g
            err['dv'][b, :, c] += (P * (eQ + up + G * rows * U32)).T @ g.abs()
            if bias is not None:
                eB = eD + (n + 16) * U32 * dS.abs()
                for i in range(bias.shape[0]):
                    val['dbias'][i, h] += dS[bucket == i].sum()
                    err['dbias'][i, h] += eB[bucket == i].sum()
    if dout is not None:
        for n in ('dk', 'dv'):
            err[n] += u * val[n].abs()
    return {n: (val[n], err[n]) for n in names}
