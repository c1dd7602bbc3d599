"""Paged serving restated on the CPU in 64 bits: append, attention, page
bookkeeping and sampling, each written from its definition with plain loops."""

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # relative half unit in the last place


def rotate(x, inv_freq, position, interleaved, factor=1.0):
    """x [tokens, heads, head_dim] rotated in 64 bits."""

    x = x.double().clone()
    half = inv_freq.numel()
    angle = position.double()[:, None, None] * inv_freq.double()
    cos, sin = factor * torch.cos(angle), factor * torch.sin(angle)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (
        slice(0, half), slice(half, 2 * half))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * cos - b * sin, b * cos + a * sin
    return x


def attention(q, k_pages, v_pages, table, lengths, scale):
    """(out, lse, weight): weight = sum_j p_j |v_j|, the scale of out's rounding."""

    n, hq, d = q.shape
    _, hk, page, _ = k_pages.shape
    out = torch.zeros((n, hq, d), dtype=torch.float64)
    weight = torch.zeros_like(out)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    size = torch.zeros((n, hq), dtype=torch.float64)  # largest sum_d |q_d k_d| * scale
    for b in range(n):
        length = int(lengths[b])
        if length == 0:
            continue
        held = table[b, :-(-length // page)].long()
        for h in range(hq):
            k = k_pages[held, h // (hq // hk)].double().reshape(-1, d)[:length]
            v = v_pages[held, h // (hq // hk)].double().reshape(-1, d)[:length]
            s = scale * (k @ q[b, h].double())
            size[b, h] = abs(scale) * (k.abs() @ q[b, h].double().abs()).max()
            lse[b, h] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[b, h])
            out[b, h], weight[b, h] = p @ v, p @ v.abs()
    return out, lse, weight, size


def cancelling_case(dtype, head_dim, group, lengths, page):
    """(q, k_pages, v_pages, table, lengths) of one KV head whose outputs nearly vanish although
    their terms do not: an error of the softmax weights stands out of the outputs' own rounding.

    Scores (at a scale of 1) are 0 at even positions and -a_h at odd ones, exact in any
    arithmetic; the weights there are 1 and e^-a_h. Values are 1 at odd positions and, at even
    ones, -e^-a_h rounded to the type, for head h = dimension modulo the group."""

    a = (0.15 + 2.7 * torch.arange(group, dtype=torch.float64) / group).to(dtype)
    counts = [-(-n // page) for n in lengths]
    pages, width = sum(counts) + 1, max(counts)
    q = torch.zeros((len(lengths), group, head_dim), dtype=dtype)
    q[:, :, 0] = a
    k = torch.randn((pages, 1, page, head_dim), generator=torch.Generator().manual_seed(2)).to(dtype)
    v = torch.empty_like(k)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    near = torch.exp(-a.double()).to(dtype)[torch.arange(head_dim) % group]
    first = 0
    for b, n in enumerate(lengths):
        for j in range(counts[b] * page):
            at = pages - 1 - first - j // page
            table[b, j // page] = at
            k[at, 0, j % page, 0] = -(j % 2)
            v[at, 0, j % page] = 1.0 if j % 2 else -near
        first += counts[b]
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32)


def cancelling_bound(dtype, want, weight, lengths):
    """What such an output may be off by: its own rounding (u |o|, 2^-25 among fp16's subnormals), weights
    in two parts of the type (u^2), the 32-bit exponent's argument (6 at most, 10 more where fp16's weights
    are lifted: 2^-19 in all) and the 32-bit sums of two products per position and of the weights."""

    u = UNIT[dtype]
    sums = (3 * lengths.double() + 16)[:, None, None] * 2.0 ** -23
    return 1.01 * u * want.abs() + (1.01 * u * u + 2.0 ** -19 + sums) * weight + 2.0 ** -25


def attention_in_parts(q, k_pages, v_pages, table, lengths, parts):
    """The outputs at a scale of 1 with weights held as `parts` values of q's type, else in 64 bits."""

    out = torch.zeros(q.shape, dtype=torch.float64)
    page = k_pages.shape[2]
    for b, length in enumerate(lengths.tolist()):
        held = table[b, :-(-length // page)].long()
        k, v = (x[held, 0].double().reshape(-1, q.shape[2])[:length] for x in (k_pages, v_pages))
        p = torch.exp(q[b].double() @ k.t())
        p = p / p.amax(-1, keepdim=True)
        kept = torch.zeros_like(p)
        for _ in range(parts):
            kept += (p - kept).to(q.dtype).double()
        out[b] = kept @ v / p.sum(-1, keepdim=True)
    return out


class Pages:
    """The bookkeeping on Python lists, page contents included: content[p] is
    any value that stands for page p."""

    def __init__(self, table, lengths, ref, content, page):
        self.table, self.lengths, self.ref, self.content = table, lengths, ref, content
        self.page = page

    def count(self, length):
        return -(-length // self.page)

    def take(self):
        page = self.ref.index(0)
        self.ref[page] = 1
        return page

    def free(self, slots):
        for s in slots:
            for j, page in enumerate(self.table[s]):
                if self.lengths[s] and page >= 0:
                    self.ref[page] -= 1
                    self.table[s][j] = -1
            self.lengths[s] = 0

    def fork(self, parents, children):
        n = len(self.lengths)
        ok = all(0 <= s < n for s in parents + children)
        if not ok or len(set(children)) < len(children) or set(children) & set(parents) or any(
                self.lengths[c] for c in children):
            return -1
        tails = [(p, c) for p, c in zip(parents, children) if self.lengths[p] % self.page]
        free = self.ref.count(0)
        if free < len(tails):
            return len(tails) - free
        for p, c in tails:
            page = self.take()
            full = self.lengths[p] // self.page
            self.table[c][full] = page
            self.content[page] = self.content[self.table[p][full]]
        for p, c in zip(parents, children):
            for j in range(self.lengths[p] // self.page):
                self.table[c][j] = self.table[p][j]
                self.ref[self.table[p][j]] += 1
            self.lengths[c] = self.lengths[p]
        return 0

    def reserve(self, extra):
        width = len(self.table[0])
        if any(e < 0 or self.count(length + e) > width for length, e in zip(self.lengths, extra)):
            return -1
        need = sum(self.count(length + e) - self.count(length) for length, e in zip(self.lengths, extra))
        free = self.ref.count(0)
        if free < need:
            return need - free
        for s, e in enumerate(extra):
            for j in range(self.count(self.lengths[s]), self.count(self.lengths[s] + e)):
                self.table[s][j] = self.take()
            self.lengths[s] += e
        return 0

    def compact(self):
        live = sum(1 for r in self.ref if r)
        holes = [i for i in range(live) if self.ref[i] == 0]
        movers = [i for i in range(live, len(self.ref)) if self.ref[i]]
        to = dict(zip(movers, holes))
        for source, target in to.items():
            self.ref[target], self.ref[source] = self.ref[source], 0
            self.content[target] = self.content[source]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live


def sample_order(logits):
    """Indexes by larger logit, then smaller index (NaN as -inf), and the logits in 64 bits."""

    x = torch.where(torch.isnan(logits.float()), -math.inf, logits.float()).double()
    return torch.sort(x, descending=True, stable=True).indices, x


def sample_check(logits, temperature, top_k, top_p, min_p, uniform, token, logprob, slack):
    """None if `token` (with `logprob`) is an answer for some thresholds within `slack` of
    the given ones (a share of the mass), else what is wrong."""

    order, x = sample_order(logits)
    top = float(x[order[0]])
    if top == -math.inf:
        return None if token == -1 and logprob == -math.inf else "an empty row must give -1"
    most = x.numel() if not top_k or top_k <= 0 else min(top_k, x.numel())
    if not temperature > 0:
        most = 1
        temperature = 1.0
    odds = torch.exp(torch.where(x == top, 0.0, (x - top) / temperature))
    ranked = order[:most]
    mass = odds[ranked]
    before = torch.cumsum(mass, 0) - mass
    share = max(0.0, top_p)
    sure = (before < (share - slack) * mass.sum()) & (mass >= min_p * (1 + slack))
    maybe = (before < (share + slack) * mass.sum()) & (mass >= min_p * (1 - slack))
    if share >= 1:
        sure, maybe = mass >= min_p * (1 + slack), mass >= min_p * (1 - slack)
    sure[0] = maybe[0] = True
    maybe = maybe | (mass == mass[0])
    if token not in ranked[maybe].tolist():
        return "token {} is not among the kept ones".format(token)
    failures = []
    for kept in (sure, maybe):
        index, where = torch.sort(ranked[kept])
        m = mass[kept][where]
        total = float(m.sum())
        at = (index == token).nonzero()
        if at.numel() == 0:
            continue
        end = float(m[:int(at) + 1].sum()) / total
        start = end - float(m[int(at)]) / total
        want = math.log(float(m[int(at)]) / total) if m[int(at)] > 0 else -math.inf
        if not start - slack <= uniform <= end + slack:
            failures.append("u={} is outside [{}, {})".format(uniform, start, end))
        elif abs(logprob - want) > 4 * slack * (1 + abs(want)):
            failures.append("log probability {} instead of {}".format(logprob, want))
        else:
            return None
    return "; ".join(failures) or "token {} is not among the kept ones".format(token)
