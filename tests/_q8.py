"""Inputs, 64-bit oracles and error bounds for the 8-bit cache tests."""

import collections
import math

import torch

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def make_cache(units, h, rows, d, block, code, seed=0):
    """Random codes and scales (the values' size differs by block and head)."""
    g = torch.Generator().manual_seed(seed)
    bits = torch.randint(0, 256, (units, h, rows, d), generator=g, dtype=torch.int32)
    if code == "e4m3":
        bits = torch.where((bits & 0x7F) == 0x7F, bits & 0x80, bits)  # no NaN
        bits = torch.where((bits & 0x78) > 0x48, bits & 0xCF, bits)   # magnitudes of a few units
    cache = bits.to(torch.uint8).view(CODES[code])
    top = 1 / 64 if code == "int8" else 1 / 2
    scale = top * torch.exp(0.7 * torch.randn(units, h, -(-rows // block), generator=g))
    return cache, scale


def values64(cache, scale, block):
    s = scale.double().repeat_interleave(block, dim=-1)[..., :cache.shape[-2]]
    return cache.float().double() * s[..., None]


def rotate64(x, cos, sin, pos):
    """x (..., T, D) float64, token t at pos + t (left as it is outside the table)."""
    out = x.clone()
    half = x.shape[-1] // 2
    for t in range(x.shape[-2]):
        if 0 <= pos + t < cos.shape[0]:
            c, s = cos[pos + t].double(), sin[pos + t].double()
            a, b = x[..., t, :half], x[..., t, half:]
            out[..., t, :half] = a * c[:half] - b * s[:half]
            out[..., t, half:] = b * c[half:] + a * s[half:]
    return out


def attention64(q, kc, vc, ks, vs, block, lens, q_lens, table, causal, scale, splits=1, dtype=None,
                rotated=False):
    """(output, bound) in float64 on the CPU.  The bound counts, for each output
    element o = sum p_n t_n c_n (u: half a step, relative, of q's type):

    * the result's rounding, u |o| (and 2^-25 where fp16 results are subnormal);
    * the probabilities' rounding to fp16, 2^-11 p_n each, or to the sum of two fp16
      numbers for fp32 queries, 2^-22 (the second one's 2^-11 of the first one's
      2^-11), and at least 2^-25 of the largest p_j t_j, the step of subnormals in
      the kernel's units;
    * the queries' rounding in the same way (rotated 16-bit ones, all fp32 ones; the
      others are exact down to 2^-25 of their row's largest element), which moves a
      score by as much of sum |q_d| |k_d| and a probability by twice that;
    * the fp32 scores: D + 16 roundings of the product's sum and a few of the
      exponent, 2^-23 each, likewise; and the fp32 sums over the keys.
    """
    b, hq, sq, d = q.shape
    hkv = kc.shape[1]
    dtype = q.dtype if dtype is None else dtype
    u = U[dtype]
    two = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    u_q = two if rotated or dtype == torch.float32 else 0.0
    out = torch.zeros(b, hq, sq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(b):
        n, m = lens[i], q_lens[i]
        if table is None:
            k, c = values64(kc[i], ks[i], block)[:, :n], vc[i].float().double()[:, :n]
            t = vs[i].double().repeat_interleave(block, dim=-1)[:, :n]
            at = torch.arange(n)
        else:
            page = kc.shape[2]
            at, ku, cu, tu = [], [], [], []
            for j in range(n):
                p, r = table[i][j // page], j % page
                if 0 <= p < kc.shape[0]:
                    at.append(j)
                    ku.append(kc[p, :, r].float().double() * ks[p, :, r // block].double()[:, None])
                    cu.append(vc[p, :, r].float().double())
                    tu.append(vs[p, :, r // block].double())
            if not at:
                continue
            at = torch.tensor(at)
            k, c, t = torch.stack(ku, 1), torch.stack(cu, 1), torch.stack(tu, 1)
        if n == 0 or m == 0:
            continue
        for h in range(hq):
            g = h // (hq // hkv)
            x = q[i, h, :m].double()
            s = x @ k[g].T * scale
            mag = (x.abs() @ k[g].abs().T * abs(scale)).amax(-1, keepdim=True)
            edge = x.abs().amax(-1, keepdim=True) * k[g].abs().sum(-1).amax() * abs(scale)
            if causal:
                s = s.masked_fill(at[None] > torch.arange(n - m, n)[:, None], -math.inf)
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            w = p * t[g]
            o, mean = w @ c[g], w @ c[g].abs()
            rel = (two + 2 * ((u_q + (d + 16) * 2.0 ** -23) * mag + 2.0 ** -25 * edge + 2.0 ** -21)
                   + (n + splits) * 2.0 ** -23)
            out[i, h, :m] = o
            tol[i, h, :m] = (rel * mean + u * o.abs() + 1e-30
                             + 2.0 ** -25 * w.amax(-1, keepdim=True) * c[g].abs().sum(0))
            if dtype == torch.float16:
                tol[i, h, :m] += 2.0 ** -25
    return out, tol


def check_within(got, want, tol):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} outside their bound, the first at {i}: "
                             f"{got[i].item()} for {want[i].item()}, bound {tol[i].item():.2e}")


class PlanModel:
    """Page bookkeeping with a queue and lists, one row at a time."""

    def __init__(self, page_size, width, max_new):
        self.page, self.width, self.max_new = page_size, width, max_new

    def step(self, pages, lens, news, free):
        """pages: list of page lists (changed); free: deque (changed).  Returns (slots,
        lens)."""
        asked, stock, given, out, slots = 0, len(free), [], [], []
        for b, n in enumerate(lens):
            d = min(news[b], self.max_new)
            row = [-1] * self.max_new
            if d < 0:
                n = max(n + d, 0)
                keep = math.ceil(n / self.page)
                given += pages[b][keep:]
                del pages[b][keep:]
            elif d > 0 and n + d <= self.width * self.page:
                want = math.ceil((n + d) / self.page) - len(pages[b])
                asked += want
                if want == 0 or asked <= stock:
                    pages[b] += [free.popleft() for _ in range(want)]
                    for t in range(d):
                        p = pages[b][(n + t) // self.page]
                        row[t] = p * self.page + (n + t) % self.page if p >= 0 else -1
                    n += d
            out.append(n)
            slots.append(row)
        free.extend(given)
        return slots, out


def random_plan(b, width, page, max_new, spare, seed):
    """A consistent state of a server: (pages, lens, news, free queue, head, ring size)."""
    g = torch.Generator().manual_seed(seed)

    def ints(lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=g).tolist()

    lens = ints(0, width * page, b)
    for i, n in enumerate((0, page, width * page, 1)[:b]):
        lens[i] = n
    total = sum(-(-n // page) for n in lens) + spare
    ids = torch.randperm(total, generator=g).tolist()
    pages, at = [], 0
    for n in lens:
        k = -(-n // page)
        pages.append(ids[at:at + k])
        at += k
    news = [x if r < 7 else -x for x, r in zip(ints(0, max_new + 2, b), ints(0, 9, b))]
    for i in range(0, b, 5):
        news[i] = -ints(0, width * page, 1)[0]
    return pages, lens, news, collections.deque(ids[at:]), total // 3, max(total, 1)


def plan_tensors(pages, free, head, size, width, device):
    """(block_table, free_pages, free_state) of that state, garbage where unused."""
    table = torch.full((len(pages), width), -7, dtype=torch.int32)
    for b, row in enumerate(pages):
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    ring = torch.full((size,), -9, dtype=torch.int32)
    for i, p in enumerate(free):
        ring[(head + i) % size] = p
    return (table.to(device), ring.to(device),
            torch.tensor([head, len(free)], dtype=torch.int32, device=device))


def check_plan(table, ring, state, slots, lens, want_pages, want_slots, want_lens, want_free):
    assert slots.dtype == torch.int64 and slots.cpu().tolist() == want_slots
    assert lens.dtype == torch.int32 and lens.cpu().tolist() == want_lens
    t, r = table.cpu().tolist(), ring.cpu().tolist()
    head, count = state.cpu().tolist()
    for row, pages in zip(t, want_pages):
        assert row[:len(pages)] == pages
    assert [r[(head + i) % len(r)] for i in range(count)] == list(want_free)
