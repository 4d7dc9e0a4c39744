"""GPU tier: every form in which lvb_attention_paged runs (clusters, whole items, dealt blocks with a join, key
ranges, a prefix in front or in a pass of its own), each with V that shows any block which is missing, read
twice or taken from elsewhere, and with lists that are wrong; and the order of append and attention on a
stream and in a graph.

Tolerance, per element, from the kernels' arithmetic (u = half a step of the type, 2^-8 bf16, 2^-11 fp16):
  u·(Σ p|V| + |O|)        P and O, rounded once each
  2^-31·Σ|V| / Σ 2^(s-max) + 2^-25   fp16: weights among the subnormals (held 2^6 above their value), and O's
  2^-14·Σ p|V|            a score's error in fp32 (sums of D products, |s| below 10) and exp2
  n·2^-27·Σ p|V|          n/16 additions of 2^-23 each in the fp32 sums over the keys
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}

# name: Hq, Hkv, page, lengths, rows per sequence, prefix, places of the table beyond the longest length;
# kernel, prefix in a pass of its own, clusters, launches
FORMS = {
    "decoding, clusters": (8, 2, 16, [700, 90, 300], 2, 0, 0, "decode", False, True, 1),
    "decoding, one CTA an item": (16, 8, 8, [500, 129, 0, 77] * 4, 1, 0, 0, "decode", False, True, 1),
    "decoding, whole items": (16, 8, 32, [500, 129, 0, 900] * 8, 1, 0, 0, "decode", False, False, 1),
    "decoding, dealt": (12, 4, 64, [20000, 3000, 1, 9000], 3, 0, 50000, "decode", False, False, 2),
    "decoding, prefix in front, clusters": (8, 2, 16, [40, 700, 3], 1, 900, 0, "decode", False, True, 1),
    "decoding, prefix in front, whole items": (8, 8, 32, [100, 60, 0, 129] * 6, 2, 600, 0, "decode", False, False, 1),
    "decoding, prefix gathered": (32, 8, 48, [100, 3000, 1, 0, 700], 1, 9000, 50000, "decode", True, False, 3),
    "flash, whole tiles": (8, 8, 64, [300, 900, 50, 129] * 3, 40, 0, 0, "flash", False, False, 1),
    "flash, more items than CTAs": (16, 8, 16, [300, 900, 150, 129] * 5, 140, 0, 0, "flash", False, False, 1),
    "flash, clusters": (8, 2, 128, [2000], 17, 0, 0, "flash", False, True, 1),
    "flash, ranges joined from memory": (8, 2, 64, [20000, 3000], 30, 0, 50000, "flash", False, None, 2),
    "flash, prefix in front": (32, 8, 24, [400, 200, 333] * 4, 100, 1000, 0, "flash", False, False, 1),
    "flash, prefix gathered": (64, 8, 32, [300, 0, 150, 20] * 8, 4, 8000, 0, "flash", True, False, 3),
    "flash, prefix gathered, own ranges": (24, 8, 64, [1500, 60, 7] * 3, 9, 8193, 0, "flash", True, False, 3),
}


class Batch:
    """A form's cache, lists and queries. `values`: what V holds, of (place, KV heads, D)."""

    def __init__(self, lvb, torch, form, T, D, values=None, seed=0):
        (self.Hq, self.Hkv, self.page, self.lens, self.q, self.prefix, more, kernel, gathered, clusters,
         launches) = FORMS[form]
        self.torch, self.lvb, self.T, self.D = torch, lvb, T, D
        dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[T]
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        B, page = len(self.lens), self.page
        counts = [-(-n // page) for n in self.lens]
        pp = -(-self.prefix // page)
        self.num_pages = sum(counts) + pp + 3
        order = torch.randperm(self.num_pages, generator=g, device="cuda").to(torch.int32)
        self.width = max(counts) + more // page
        self.table = torch.full((B, self.width), -7, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.prefix_table = order[at:at + pp].contiguous()
        shape = (self.num_pages, page, self.Hkv, D)
        self.Kc, self.Vc = (torch.full(shape, float("nan"), dtype=dt, device="cuda") for _ in "kv")
        for row, n, first in [(self.prefix_table, self.prefix, 0)] + [
                (self.table[b], n, self.prefix) for b, n in enumerate(self.lens)]:
            p = torch.arange(n, device="cuda")
            where = row.long()[p // page], p % page
            self.Kc[where] = torch.randn(n, self.Hkv, D, device="cuda", generator=g).to(dt)
            self.Vc[where] = (torch.randn(n, self.Hkv, D, device="cuda", generator=g).to(dt) if values is None
                              else values(p + first, self.Hkv, D).to(dt))
        self.tokens = self.q * B + 2
        self.cu = [self.q * b for b in range(B + 1)]
        self.Q = torch.randn(self.tokens, self.Hq, D, device="cuda", generator=g).to(dt)
        p = lvb.attention_paged_plan(B, self.Hq, self.Hkv, self.tokens, self.q, page, self.width, D=D,
                                     prefix_len=self.prefix)
        assert (p.kernel, p.prefix_splits > 0, p.launches) == (
            {"decode": lvb.PAGED_DECODE, "flash": lvb.PAGED_FLASH}[kernel], gathered, launches), form
        assert clusters is None or (p.cluster > 0) == clusters, form

    def ints(self, x):
        return self.torch.tensor(x, dtype=self.torch.int32, device="cuda")

    def run(self, lens=None, cu=None, table=None, prefix_table=None, max_q=None):
        """O and lse (both 7 where nothing is written) and the status word."""
        torch = self.torch
        O = torch.full_like(self.Q, 7.0)
        lse = torch.full((self.tokens, self.Hq), 7.0, device="cuda")
        more = {}
        if self.prefix:
            more = dict(prefix_len=self.prefix,
                        prefix_table=self.prefix_table if prefix_table is None else prefix_table)
        self.lvb.attention_paged(O, self.Q, self.Kc, self.Vc, self.table if table is None else table,
                                 self.ints(lens or self.lens), cu_q=self.ints(cu or self.cu),
                                 max_q=max_q or self.q, lse=lse, **more)
        torch.cuda.synchronize()
        return O, lse, self.lvb.device_status()

    def keys(self, row, n):
        """K and V of places 0 .. n-1 in 64 bits; zeros where the row's page is none."""
        torch = self.torch
        p = torch.arange(n, device="cuda")
        page = row.long()[p // self.page]
        bad = ((page < 0) | (page >= self.num_pages))[:, None, None]
        page = torch.where(bad[:, 0, 0], 0, page)
        return [torch.where(bad, 0.0, c[page, p % self.page].double()) for c in (self.Kc, self.Vc)]

    def check(self, O, lse, lens=None, cu=None, table=None, prefix_table=None, max_q=None):
        """Each sequence against the definition, with what the lists get wrong limited as include/lvb.h
        says; rows of no sequence as they were."""
        torch = self.torch
        lens, cu, max_q = lens or self.lens, cu or self.cu, max_q or self.q
        table = self.table if table is None else table
        Kp, Vp = self.keys(self.prefix_table if prefix_table is None else prefix_table, self.prefix)
        left = torch.ones(self.tokens, dtype=torch.bool, device="cuda")
        G = self.Hq // self.Hkv
        for b, n in enumerate(lens):
            r0, r1 = cu[b], cu[b + 1]
            if not (0 <= r1 - r0 <= max_q and 0 <= r0 and r1 <= self.tokens):
                continue
            if not 0 <= n <= self.width * self.page:
                n = 0
            q = r1 - r0
            left[r0:r1] = False
            K, V = (torch.cat(x) for x in zip((Kp, Vp), self.keys(table[b], n)))
            x = self.Q[r0:r1].double().unflatten(1, (self.Hkv, G))
            s = torch.einsum("qhgd,nhd->hgqn", x, K) * self.D ** -0.5
            place = torch.arange(-self.prefix, n, device="cuda")
            seen = (place < 0) | (place <= (n - q + torch.arange(q, device="cuda"))[:, None])
            s = torch.where(seen, s, -torch.inf)
            m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), -torch.inf)
            w = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
            l = w.sum(-1, keepdim=True)
            p = torch.where(l > 0, w / l, 0.0)
            ref = torch.einsum("hgqn,nhd->qhgd", p, V)
            size = torch.einsum("hgqn,nhd->qhgd", p, V.abs())
            lref = (torch.where(torch.isinf(m), 0.0, m) + torch.log(l))[..., 0].permute(2, 0, 1)
            bound = U[self.T] * (size + ref.abs()) + (2.0 ** -14 + place.numel() * 2.0 ** -27) * size
            if self.T == "fp16":
                some = l.clamp(min=1.0).permute(2, 0, 1, 3)
                bound = bound + 2.0 ** -31 * V.abs().sum(0)[None, :, None] / some + 2.0 ** -25
            err = (O[r0:r1].double().unflatten(1, (self.Hkv, G)) - ref).abs()
            assert bool((err <= bound).all()), (b, n, float((err - bound).max()), float(err.max()))
            got = lse[r0:r1].double().unflatten(1, (self.Hkv, G))
            none = torch.isinf(lref)
            assert torch.equal(torch.isneginf(got), none)
            assert bool(((got - lref).abs() <= 2.0 ** -14 * (1 + lref.abs()))[~none].all()), b
        assert bool((O[left] == 7).all()) and bool((lse[left] == 7).all())


@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("form", FORMS)
def test_every_box_of_keys_counts(lvb, torch_cuda, form, T, D):
    """V is 1 in one column per run of eight places and 0 elsewhere, so that a column of O is the weight
    of its few runs. A block of 128 places that is missing, doubled or out of its place exceeds the bf16 bound
    3.5 times among 20,000 keys of 64-wide heads, 7.7 times of 128-wide ones, more among fewer keys."""
    def columns(place, Hkv, D):
        torch = torch_cuda
        c = (place[:, None] // 8 + 5 * torch.arange(Hkv, device="cuda")) % D
        return torch.nn.functional.one_hot(c, D).double()
    c = Batch(lvb, torch_cuda, form, T, D, columns, seed=1)
    O, lse, status = c.run()
    assert status == (0, 0, 0)
    c.check(O, lse)


@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("form", FORMS)
def test_wrong_lists(lvb, torch_cuda, form, T, D):
    """Lengths, pages and rows that the kernels' own checks refuse: the status word names the site, the
    sequence is limited as documented, and all others are right."""
    c = Batch(lvb, torch_cuda, form, T, D, seed=2)
    O, lse, status = c.run()
    assert status == (0, 0, 0)
    c.check(O, lse)
    B, q, long = len(c.lens), c.q, int(np.argmax(c.lens))

    def wrong(site, **kw):
        O, lse, status = c.run(**kw)
        assert status[:2] == (lvb.LVB_ERR_INVALID_ARG, site), (kw, status)
        c.check(O, lse, **kw)
    for n in (-1, -2 ** 31, c.width * c.page + 1, 2 ** 31 - 1):
        wrong(81, lens=c.lens[:long] + [n] + c.lens[long + 1:])
    for page in (-1, c.num_pages, 2 ** 31 - 1, -2 ** 31):
        table = c.table.clone()
        table[long, 0] = page
        wrong(82, table=table)
        if c.prefix:
            prefix_table = c.prefix_table.clone()
            prefix_table[-1] = page
            wrong(82, prefix_table=prefix_table)
    wrong(83, cu=c.cu[:-1] + [c.cu[-1] + 1])                            # a row more than max_q
    wrong(83, cu=c.cu[:-1] + [c.tokens + 1], max_q=q + 3)               # rows behind the last token
    wrong(83, cu=[-1, q - 1] + c.cu[2:], max_q=q + 1)                   # a row before the first
    wrong(83, cu=[q + 1] + c.cu[1:])                                    # fewer than no rows
    wrong(83, cu=[-2 ** 31] + c.cu[1:])
    wrong(83, cu=c.cu[:-1] + [2 ** 31 - 1])
    O2, lse2, status = c.run()
    assert status == (0, 0, 0) and torch_cuda.equal(O2, O) and torch_cuda.equal(lse2, lse)


@pytest.mark.parametrize("form", ["decoding, prefix gathered", "flash, prefix gathered", "decoding, dealt",
                                  "decoding, prefix in front, clusters"])
def test_append_then_attend_on_a_stream(lvb, torch_cuda, form):
    """Steps of append and attention one behind the other without a wait between them, and the same
    steps with one: the kernels that start beside the ones before them read what those wrote."""
    torch = torch_cuda
    c = Batch(lvb, torch, form, "bf16", 128, seed=3)
    B, q, steps = len(c.lens), c.q, 12
    start = [max(0, min(n, c.width * c.page - steps * q)) for n in c.lens]
    used = {int(x) for x in c.prefix_table}
    free = [x for x in range(c.num_pages) if x not in used]
    need = [-(-(n + steps * q) // c.page) for n in start]
    # pages enough for the steps: a larger cache, the old one's pages first
    extra = max(0, sum(need) - len(free))
    Kc, Vc = (torch.cat([x, torch.zeros(extra, *x.shape[1:], device="cuda", dtype=x.dtype)]).nan_to_num(0.5)
              for x in (c.Kc, c.Vc))
    free += range(c.num_pages, c.num_pages + extra)
    table = torch.zeros(B, max(c.width, max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = c.ints(free[at:at + n])
        at += n
    lens = [c.ints([n + (i + 1) * q for n in start]) for i in range(steps)]
    new = [[torch.randn(B * q, h, 128, device="cuda", generator=c.g).to(torch.bfloat16)
            for h in (c.Hkv, c.Hkv, c.Hq)] for _ in range(steps)]
    f = torch.exp(-torch.arange(64, dtype=torch.float64, device="cuda") * 0.14)
    more = dict(prefix_table=c.prefix_table, prefix_len=c.prefix) if c.prefix else {}

    def go(wait):
        cache = Kc.clone(), Vc.clone()
        O = [torch.empty(B * q, c.Hq, 128, device="cuda", dtype=torch.bfloat16) for _ in range(steps)]
        Qr = torch.empty_like(O[0])
        torch.cuda.synchronize()
        for i in range(steps):
            K, V, Q = new[i]
            lvb.kv_append(*cache, K, V, table, lens[i], max_q=q, Q=Q, Qo=Qr, freqs=f, prefix_len=c.prefix)
            if wait:
                torch.cuda.synchronize()
            lvb.attention_paged(O[i], Qr, *cache, table, lens[i], max_q=q, **more)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert lvb.device_status() == (0, 0, 0)
        return [*O, *cache]
    want = go(True)
    assert all(bool(torch.isfinite(x.float()).all()) for x in want)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, go(False)))


@pytest.mark.parametrize("form", ["decoding, prefix gathered", "flash, prefix gathered",
                                  "flash, ranges joined from memory", "flash, more items than CTAs"])
def test_captured_call(lvb, torch_cuda, form):
    """Calls of several launches with their workspaces captured into two graphs that run in turn and side
    by side, replayed while the lists, the queries and the pages change."""
    torch = torch_cuda
    c = Batch(lvb, torch, form, "fp16", 64, seed=4)
    lens, cu = c.ints(c.lens), c.ints(c.cu)
    O = [torch.full_like(c.Q, 7.0) for _ in range(2)]
    lse = [torch.full((c.tokens, c.Hq), 7.0, device="cuda") for _ in range(2)]
    more = dict(prefix_table=c.prefix_table, prefix_len=c.prefix) if c.prefix else {}
    calls = [lvb.prepare_attention_paged(o, c.Q, c.Kc, c.Vc, c.table, lens, cu_q=cu, max_q=c.q, lse=x, **more)
             for o, x in zip(O, lse)]
    streams = [torch.cuda.Stream() for _ in calls]
    graphs = []
    calls[0]()
    torch.cuda.synchronize()
    for call, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        graphs.append(g)
    for step in range(4):
        c.Q.normal_(generator=c.g)
        now = [max(0, n - 3 * step * (b % 3)) for b, n in enumerate(c.lens)]
        lens.copy_(c.ints(now))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                if step % 2 == 0:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert lvb.device_status() == (0, 0, 0)
        c.check(O[0], lse[0], lens=now)
        assert torch.equal(O[0], O[1]) and torch.equal(lse[0], lse[1])
        eager, elser, status = c.run(lens=now)
        assert status == (0, 0, 0) and torch.equal(eager, O[0]) and torch.equal(elser, lse[0])
