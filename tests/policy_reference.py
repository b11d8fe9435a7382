"""Plain restatement, in 64 bits on the CPU, of the policy operators' definitions (include/gymhip.h): what their tests compare against."""
import math

import numpy as np
import torch

LOW = 0xFFFFFFFF


def words(block, row, step, seed):
    """Philox4x32, 7 rounds, on Python integers held in object arrays: (block, row, step) -> four 32-bit words.  Unhurried and literal."""
    block, row, step = np.broadcast_arrays(np.asarray(block, object), np.asarray(row, object), np.asarray(step, object))
    c = [block & LOW, row & LOW, step & LOW, (row >> 32 & 0xFFFF) | ((step >> 32 & 0xFFFF) << 16)]
    k = [seed & LOW, seed >> 32 & LOW]
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & LOW, (a >> 32) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return c


def row_keys(n, rows=0, step=0):
    """(row keys, steps) as unsigned Python integers [n]."""
    m = 1 << 64
    r = [int(v) % m for v in rows] if isinstance(rows, torch.Tensor) else [(int(rows) + i) % m for i in range(n)]
    if isinstance(step, torch.Tensor):
        s = [int(v) % m for v in step.reshape(-1)]
        s = s * n if len(s) == 1 and n != 1 else s
    else:
        s = [int(step) % m] * n
    return np.array(r, object), np.array(s, object)


def uniforms(n, seed, rows=0, step=0):
    r, s = row_keys(n, rows, step)
    w = words(LOW, r, s, seed)
    return torch.tensor([(float((int(a) << 20) | (int(b) >> 12)) + 0.5) * 2.0 ** -52 for a, b in zip(w[0], w[1])], dtype=torch.float64)


def kept(n, width, p, seed, rows=0, step=0):
    r, s = row_keys(n, rows, step)
    w = words(np.arange((width + 7) // 8, dtype=object)[None, :], r[:, None], s[:, None], seed)
    lanes = np.stack([half for v in w for half in (v & 0xFFFF, v >> 16)], axis=-1).reshape(n, -1)[:, :width]
    return torch.from_numpy((lanes >= round(65536 * p)).astype(bool).reshape(n, width))


def column(v, n):
    v = v.detach().cpu().float() if isinstance(v, torch.Tensor) else torch.full((n,), float(v), dtype=torch.float32)
    return v.double()


def apply_rules(x, rules):
    """(z, dz/dx, greedy rows) of x [n, width], all in float64 on the CPU."""
    x = x.detach().cpu().double()
    n, width = x.shape
    z, slope = x.clone(), torch.ones_like(x)
    greedy = torch.zeros(n, dtype=torch.bool)
    if rules is None:
        return z, slope, greedy
    rep, pres, freq, temp = (column(getattr(rules, k), n) for k in ("repetition", "presence", "frequency", "temperature"))
    if rules.history is not None:
        h = rules.history.cpu()
        for b in range(n):
            count = int(rules.history_len[b]) if rules.history_len is not None else h.shape[1]
            ids = h[b, :max(0, min(count, h.shape[1]))].long()
            ids = ids[(ids >= 0) & (ids < width)]
            c = torch.bincount(ids, minlength=width).double()
            hit = c > 0
            up = x[b] > 0
            z[b] = torch.where(hit, torch.where(up, x[b] / rep[b], x[b] * rep[b]) - freq[b] * c - pres[b], x[b])
            slope[b] = torch.where(hit, torch.where(up, 1 / rep[b], rep[b]), slope[b])
    if rules.bias is not None:
        z = z + rules.bias.cpu().double()
    greedy = ~(temp > 0)
    t = torch.where(greedy, 1.0, temp)[:, None]
    z, slope = z / t, slope / t
    if rules.mask is not None:
        m = rules.mask.cpu().numpy().view(np.uint32)
        bits = torch.from_numpy(((m[:, np.arange(width) // 32] >> (np.arange(width) % 32).astype(np.uint32)) & 1).astype(bool))
        if rules.mask_rows is not None:
            lines = rules.mask_rows.cpu().tolist()
            legal = torch.stack([torch.ones(width, dtype=torch.bool) if k < 0 else torch.zeros(width, dtype=torch.bool) if k >= len(bits) else bits[k]
                                 for k in lines]) if n else torch.zeros(0, width, dtype=torch.bool)
        else:
            legal = bits.expand(n, width)
        z = torch.where(legal, z, -math.inf)
        slope = torch.where(legal, slope, 0.0)
    return z, slope, greedy


def softmax_parts(z):
    """(m, d = z - m, w = exp d, S) per row; a row without any finite or greater z has m = 0, S = 0."""
    m = z.max(1, keepdim=True).values if z.shape[1] else torch.full((z.shape[0], 1), -math.inf, dtype=z.dtype)
    base = torch.where(m == -math.inf, 0.0, m)
    d = z - base
    w = torch.exp(d)
    return base, d, w, w.sum(1, keepdim=True)


def sample(x, rules, seed, rows=0, step=0):
    z, _, greedy = apply_rules(x, rules)
    n, width = z.shape
    base, _, w, total = softmax_parts(z)
    u = uniforms(n, seed, rows, step)
    actions, lps = [], []
    for b in range(n):
        s = float(total[b])
        if not (0 < s < math.inf):
            actions.append(-1)
            lps.append(-math.inf if s == 0 else math.nan)
            continue
        if greedy[b]:
            a = int((z[b] == z[b].max()).nonzero()[0])
        else:
            upto = torch.cumsum(w[b], 0)
            a = int((upto <= float(u[b]) * float(upto[-1])).sum())
            if a >= width:
                a = int((w[b] > 0).nonzero()[-1])
        actions.append(a)
        lps.append(float(z[b, a]) - float(base[b]) - math.log(s))
    return torch.tensor(actions, dtype=torch.int32), torch.tensor(lps, dtype=torch.float64)


def score(x, actions, rules):
    """dict of log_prob, entropy (float64 [n]) and what the error bounds need."""
    z, slope, _ = apply_rules(x, rules)
    n, width = z.shape
    base, d, w, total = softmax_parts(z)
    some = total[:, 0] > 0
    p = torch.where(total > 0, w / total, 0.0)
    logs = d - torch.log(total)
    plogs = torch.where(p > 0, p * logs, 0.0)
    entropy = torch.where(some, -plogs.sum(1), 0.0)
    entropy = torch.where(torch.isnan(total[:, 0]), math.nan, entropy)
    a = actions.cpu().long()
    inside = (a >= 0) & (a < width)
    taken = logs.gather(1, a.clamp(0, max(0, width - 1))[:, None])[:, 0] if width else torch.full((n,), -math.inf, dtype=torch.float64)
    lp = torch.where(inside & ((total[:, 0] > 0) | torch.isnan(total[:, 0])), taken, -math.inf)
    return dict(z=z, slope=slope, d=d, p=p, logs=logs, entropy=entropy, log_prob=lp, some=some, inside=inside)


def score_gradient(r, actions, g_lp, g_ent):
    a = actions.cpu().long()
    n, width = r["p"].shape
    g_lp = torch.where(r["log_prob"] == -math.inf, 0.0, g_lp.cpu().double())[:, None]
    hot = torch.zeros(n, width, dtype=torch.float64)
    rows = torch.arange(n)[r["inside"]]
    hot[rows, a[r["inside"]]] = 1.0
    lp = torch.where(r["p"] > 0, r["logs"], 0.0)
    g = g_lp * (hot - r["p"]) - g_ent.cpu().double()[:, None] * r["p"] * (lp + r["entropy"][:, None])
    g = torch.where(r["some"][:, None], g, 0.0)
    return torch.where((r["slope"] == 0) | (r["z"] == -math.inf), 0.0, g * r["slope"])
