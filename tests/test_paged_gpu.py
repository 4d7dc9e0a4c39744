"""GPU tier: position rotation, the paged KV cache's append and the attention over it, through the
Python mirror against the float64 definitions (oracle/paged.py).

Tolerances, from the kernels' arithmetic (u = half a step of the type relative to the value: 2^-8
bf16, 2^-11 fp16, 2^-24 fp32):
  rotation   |Δ| <= u·|y| + 2^-21·(|x_0| + |x_1|) + 2^-25: one rounding to the type; the angle's
             fraction of a turn in fp32 (2^-25·2π < 2^-22), cos and sin within 2 units of 2^-24,
             two products and a sum (3·2^-24); half a step of fp16's subnormals.
  attention  |Δ| <= u·(max|V| + |O|) + 2^-14·max|V|: P is rounded to the type once (each weight by
             at most u), O at the store; fp32 accumulation over up to 2^12 sums of a block's 128
             keys and exp2 to 2^-22 stay below 2^-14. lse: 2^-14·(1 + |lse|) (fp32 scores).
Caches are filled with NaN wherever no token lies, tables with page numbers of no page behind a
sequence's last, so a read of either shows.
"""
import numpy as np
import pytest

from oracle.paged import attention_one, rotate

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def tdt(torch, T):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[T]


def status_ok(lvb):
    assert lvb.device_status() == (0, 0, 0)


def np64(t):
    return t.double().cpu().numpy()


def freqs_of(torch, pairs):
    return torch.exp(-torch.arange(pairs, dtype=torch.float64, device="cuda") * (9.21 / pairs))


# ---- rotation -----------------------------------------------------------------------------
def rot_bound(x, ref, pairs, layout, T):
    a = np.abs(np64(x))
    p = np.zeros_like(a)
    if layout == "halves":
        s = a[..., :pairs] + a[..., pairs:2 * pairs]
        p[..., :pairs] = p[..., pairs:2 * pairs] = s
    else:
        s = a[..., 0:2 * pairs:2] + a[..., 1:2 * pairs:2]
        p[..., 0:2 * pairs:2] = p[..., 1:2 * pairs:2] = s
    return U[T] * np.abs(ref) + 2.0 ** -21 * p + 2.0 ** -25


@pytest.mark.parametrize("T", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,pairs,sections,inverse", [
    (1, 1, 0, 1, 64, 32, None, False),            # one token, no keys
    (2, 5, 1, 37, 128, 64, None, False),          # odd counts
    (3, 4, 2, 130, 128, 48, (16, 20, 12), True),  # three axes, a rest of 32, the gradient
    (1, 3, 3, 70, 96, 24, (24, 0), False),        # an axis without a pair
    (2, 2, 1, 9, 512, 256, (100, 56, 60, 40), False),
    (1, 2, 1, 5, 16, 8, None, True),              # the smallest head
])
def test_rope(lvb, torch_cuda, T, layout, B, Hq, Hkv, S, D, pairs, sections, inverse):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(S + D)
    Q = torch.randn(B, Hq, S, D, device="cuda", generator=g).to(tdt(torch, T))
    K = torch.randn(B, Hkv, S, D, device="cuda", generator=g).to(tdt(torch, T)) if Hkv else None
    axes = len(sections) if sections else 1
    pos = torch.randint(-5, 2 ** 24 if S == 70 else 120000, (axes, B, S), device="cuda",
                        dtype=torch.int32, generator=g)
    f = freqs_of(torch, pairs)
    Qo, Ko = torch.empty_like(Q), torch.empty_like(K) if Hkv else None
    lvb.rope(Qo, Q, pos if axes > 1 else pos[0], f, Ko=Ko, K=K, sections=sections, layout=layout,
             inverse=inverse)
    for x, y in ((Q, Qo), (K, Ko)):
        if x is None:
            continue
        p = pos.cpu().numpy()[:, :, None, :]
        ref = rotate(np64(x), p, f.cpu().numpy(), list(sections) if sections else None, layout, inverse)
        assert (np.abs(np64(y) - ref) <= rot_bound(x, ref, pairs, layout, T)).all()
        assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])
    status_ok(lvb)


def test_rope_strides_in_place_and_shared_positions(lvb, torch_cuda):
    """Q and K as slices of one [B][S][H][D] projection, rotated in place with positions that all
    sequences share; what lies beside them stays."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(2, 33, 10, 128, device="cuda", generator=g).to(torch.bfloat16)
    was = qkv.clone()
    Q, K = qkv[:, :, :6].transpose(1, 2), qkv[:, :, 6:8].transpose(1, 2)
    pos = torch.arange(33, device="cuda", dtype=torch.int32)[None] * 1000
    f = freqs_of(torch, 64)
    lvb.rope(Q, Q, pos, f, Ko=K, K=K)
    ref = rotate(np64(was[:, :, :8].transpose(1, 2)), pos.cpu().numpy()[None, :, None], f.cpu().numpy())
    got = np64(qkv[:, :, :8].transpose(1, 2))
    assert (np.abs(got - ref) <= rot_bound(was[:, :, :8].transpose(1, 2), ref, 64, "halves", "bf16")).all()
    assert torch.equal(qkv[:, :, 8:], was[:, :, 8:])
    status_ok(lvb)


def test_rope_gradient(lvb, torch_cuda):
    """The inverse is the gradient: against autograd of the plain formula in float64, and against
    differences of the forward pass along a direction (the rotation is linear in x, so a
    difference of any size is exact but for rounding)."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 3, 17, 64, device="cuda", generator=g)
    w = torch.randn(2, 3, 17, 64, device="cuda", generator=g)     # gradient of the result
    v = torch.randn(2, 3, 17, 64, device="cuda", generator=g)     # direction
    pos = torch.randint(0, 50000, (3, 2, 17), device="cuda", dtype=torch.int32, generator=g)
    f, sec = freqs_of(torch, 32), (8, 12, 12)
    dx = torch.empty_like(x)
    lvb.rope(dx, w, pos, f, sections=sec, inverse=True)
    x64 = x.double().requires_grad_()
    axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(sec, device="cuda"))
    a = pos[axis].movedim(0, -1).double()[:, None] * f
    y = torch.cat([x64[..., :32] * a.cos() - x64[..., 32:] * a.sin(),
                   x64[..., 32:] * a.cos() + x64[..., :32] * a.sin()], -1)
    (y * w.double()).sum().backward()
    assert (dx.double() - x64.grad).abs().max() <= 2.0 ** -20 * 2 * w.abs().max()
    y0, y1 = torch.empty_like(x), torch.empty_like(x)
    lvb.rope(y0, x, pos, f, sections=sec)
    lvb.rope(y1, x + v, pos, f, sections=sec)
    along = ((y1 - y0).double() * w.double()).sum()
    want = (dx.double() * ((x + v) - x).double()).sum()
    n = x.numel()
    assert abs(float(along - want)) <= n ** 0.5 * 2.0 ** -18 * float(w.abs().max()) * 8


# ---- the paged cache ------------------------------------------------------------------------
class Cache:
    """A paged cache of a batch: pages dealt at random, NaN where no token lies."""

    def __init__(self, torch, T, Hkv, D, page, lens, prefix=0, spare=3, seed=0, head_major=False,
                 width_more=2):
        self.torch, self.page, self.lens, self.prefix = torch, page, list(lens), prefix
        self.T = T
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        dt = tdt(torch, T)
        pages = [-(-n // page) for n in lens]
        pp = -(-prefix // page)
        total = sum(pages) + pp + spare
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        width = max(pages + [1]) + width_more
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.prefix_table = order[at:at + pp].contiguous()
        self.spare = order[at + pp:].tolist()
        shape = (total, Hkv, page, D) if head_major else (total, page, Hkv, D)
        self.Kc, self.Vc = (torch.full(shape, float("nan"), dtype=dt, device="cuda") for _ in "kv")
        if head_major:
            self.Kc, self.Vc = self.Kc.transpose(1, 2), self.Vc.transpose(1, 2)
        self.K = [torch.randn(n, Hkv, D, device="cuda", generator=g).to(dt) for n in lens]
        self.V = [torch.randn(n, Hkv, D, device="cuda", generator=g).to(dt) for n in lens]
        self.Kp, self.Vp = (torch.randn(prefix, Hkv, D, device="cuda", generator=g).to(dt) for _ in "kv")
        for b, n in enumerate(lens):
            self.put(self.table[b], self.K[b], self.V[b])
        self.put(self.prefix_table, self.Kp, self.Vp)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def put(self, row, K, V):
        p = self.torch.arange(K.shape[0], device="cuda")
        pages, slots = row.long()[p // self.page], p % self.page
        self.Kc[pages, slots] = K
        self.Vc[pages, slots] = V


def cu_of(torch, qlens):
    return torch.tensor(np.concatenate([[0], np.cumsum(qlens)]), dtype=torch.int32, device="cuda")


def check_attention(c, Q, O, lse, qlens, causal, scale):
    Qn, On = np64(Q), np64(O)
    ln = lse.cpu().numpy().astype(np.float64)
    Hkv = c.Kc.shape[2]
    g = Q.shape[1] // Hkv
    t = 0
    Kp, Vp = np64(c.Kp), np64(c.Vp)
    for b, n in enumerate(c.lens):
        K, V = np.concatenate([Kp, np64(c.K[b])]), np.concatenate([Vp, np64(c.V[b])])
        rows = slice(t, t + qlens[b])
        for h in range(Hkv):
            ref, lref = attention_one(Qn[rows, h * g:(h + 1) * g], K[:, h], V[:, h], n, qlens[b],
                                      c.prefix, causal, scale)
            got, lgot = On[rows, h * g:(h + 1) * g], ln[rows, h * g:(h + 1) * g]
            mv = np.abs(V[:, h]).max(initial=0)
            bound = U[c.T] * (mv + np.abs(ref)) + 2.0 ** -14 * mv
            assert (np.abs(got - ref) <= bound).all(), (b, h, np.abs(got - ref).max(), bound.max())
            inf = np.isinf(lref)
            assert np.array_equal(np.isneginf(lgot), inf)
            assert (np.abs(lgot - lref)[~inf] <= 2.0 ** -14 * (1 + np.abs(lref[~inf]))).all()
        t += qlens[b]


def run_attention(lvb, torch, c, Hq, qlens, causal=True, scale=None, cu=True, spare_rows=0, Q=None,
                  max_q=None):
    D = c.Kc.shape[3]
    T = sum(qlens) + spare_rows
    if Q is None:
        Q = torch.randn(T, Hq, D, device="cuda", generator=c.g).to(c.Kc.dtype)
    O = torch.full((T, Hq, D), 7.0, device="cuda", dtype=Q.dtype)
    lse = torch.full((T, Hq), 7.0, device="cuda")
    more = dict(prefix_table=c.prefix_table, prefix_len=c.prefix) if c.prefix else {}
    lvb.attention_paged(O, Q, c.Kc, c.Vc, c.table, c.seq_lens, cu_q=cu_of(torch, qlens) if cu else None,
                        max_q=max_q or max(qlens), causal=causal, scale=scale, lse=lse, **more)
    torch.cuda.synchronize()
    status_ok(lvb)
    n = sum(qlens)
    assert bool((O[n:] == 7).all()) and bool((lse[n:] == 7).all())
    check_attention(c, Q[:n], O[:n], lse[:n], qlens, causal, scale or D ** -0.5)
    return Q, O, lse


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("page,Hq,Hkv,lens,qlens,causal", [
    (16, 1, 1, [1], [1], True),                                   # one key
    (16, 32, 8, [3000], [1], True),                               # one sequence over all SMs
    (8, 8, 8, [1, 7, 8, 9, 127, 128, 129, 700], [1] * 8, True),   # ends around a page and a block
    (64, 64, 8, [0, 1000, 64, 0, 3], [1] * 5, True),              # sequences without a key
    (48, 12, 4, [500, 2, 131], [3, 1, 2], True),                  # pages that no block divides
    (256, 16, 1, [300, 5000], [1, 1], True),                      # 16 rows per KV head
    (32, 8, 2, [77, 1, 260], [4, 2, 0], True),                    # rows that see no key, no rows
    (16, 12, 4, [90, 300], [5, 5], False),                        # no causal mask
    (24, 6, 2, [20000], [2], True),                               # one long sequence: split
    (128, 4, 4, [3000, 40, 2500, 1, 900, 128, 129] * 5, [1] * 35, True),
    (16, 8, 8, [900, 40, 0, 1, 500, 128, 129, 257] * 9, [1, 2, 1, 1, 0, 2, 1, 2] * 9, True),   # whole items
])
def test_decode(lvb, torch_cuda, T, D, page, Hq, Hkv, lens, qlens, causal, wide):
    """With a table as wide as the lengths (short or few sequences: clusters of CTAs join an item in
    shared memory) and with one for 100,000 keys (the blocks are dealt to all CTAs)."""
    c = Cache(torch_cuda, T, Hkv, D, page, lens, seed=page + Hq, width_more=100000 // page if wide else 2)
    plan = lvb.attention_paged_plan(len(lens), Hq, Hkv, sum(qlens), max(qlens), page, c.table.shape[1], D=D)
    assert plan.kernel == lvb.PAGED_DECODE
    if wide:
        assert plan.cluster == 0
    run_attention(lvb, torch_cuda, c, Hq, qlens, causal, spare_rows=2)


@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("page,Hq,Hkv,lens,qlens,causal", [
    (16, 8, 1, [40], [5], True),                          # 40 rows of one tile
    (256, 32, 1, [300, 5000], [1, 1], True),              # 32 rows of a token
    (32, 16, 2, [77, 1, 260], [4, 2, 0], True),           # rows that see no key, no rows
    (16, 16, 4, [90, 300], [5, 5], False),                # 20 rows, no causal mask
    (64, 2, 2, [256, 300], [256, 40], True),              # one head per KV head
    (8, 6, 2, [700, 0, 333, 130], [200, 0, 333, 1], True),   # groups of 3: 42 positions a tile
    (48, 10, 2, [1000, 90], [130, 80], True),             # groups of 5
    (32, 36, 1, [100, 640, 2], [7, 300, 2], True),        # groups of 36: 3 positions a tile
    (16, 128, 1, [300], [3], True),                       # 128 heads on one KV head
    (128, 4, 2, [50, 200], [90, 100], True),              # more rows than keys: rows without a key
    (64, 8, 2, [500, 129], [100, 129], False),            # no causal mask
    (256, 4, 1, [9000], [33], True),                      # a small chunk over a long cache: split
])
def test_chunks(lvb, torch_cuda, T, D, page, Hq, Hkv, lens, qlens, causal):
    assert lvb.attention_paged_plan(len(lens), Hq, Hkv, sum(qlens), max(qlens), page, 9,
                                    D=D).kernel == lvb.PAGED_FLASH
    c = Cache(torch_cuda, T, Hkv, D, page, lens, seed=page + Hq)
    run_attention(lvb, torch_cuda, c, Hq, qlens, causal, spare_rows=1)


@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("page,Hq,Hkv,prefix,lens,qlens,cluster", [
    (16, 4, 1, 1, [1], [1], True),                              # one block of each
    (8, 8, 8, 129, [0, 7, 300, 0], [1, 2, 1, 0], True),         # none of their own; no rows
    (48, 12, 2, 700, [500, 2, 131], [2, 1, 2], True),           # runs that pass from one to the other
    (64, 16, 1, 2600, [900, 64], [1, 1], True),
    (32, 8, 8, 255, [40, 0, 1, 128, 129, 257, 300] * 4, [2, 1, 1, 1, 2, 0, 2] * 4, False),   # whole items
    (32, 16, 8, 896, [33, 1, 0] * 8, [1] * 24, False),
])
def test_prefix_in_front(lvb, torch_cuda, T, D, page, Hq, Hkv, prefix, lens, qlens, cluster):
    """Few or short sequences: the decoding kernel reads the prefix in front of each one's own keys."""
    c = Cache(torch_cuda, T, Hkv, D, page, lens, prefix=prefix, seed=prefix)
    p = lvb.attention_paged_plan(len(lens), Hq, Hkv, sum(qlens) + 2, max(qlens), page, c.table.shape[1], D=D,
                                 prefix_len=prefix)
    assert (p.kernel, p.prefix_splits, p.launches, p.cluster > 0) == (lvb.PAGED_DECODE, 0, 1, cluster)
    run_attention(lvb, torch_cuda, c, Hq, qlens, spare_rows=2)
    run_attention(lvb, torch_cuda, c, Hq, qlens, causal=False)


@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("page,Hq,Hkv,prefix,lens,qlens", [
    (16, 1, 1, 1, [1], [1]),
    (16, 32, 8, 500, [1, 40, 7, 64], [1] * 4),            # one tile of rows, a page that ends inside
    (64, 8, 8, 4099, [0, 3, 300], [1, 3, 2]),             # a sequence without own keys
    (32, 64, 8, 1024, [33] * 40, [1] * 40),               # several tiles of rows
    (8, 16, 2, 129, [200, 900, 1], [4, 4, 1]),
    (64, 8, 2, 300, [400, 50, 0], [200, 50, 12]),         # chunks behind a prefix: flash
    (48, 4, 4, 128, [300], [300]),
])
def test_shared_prefix(lvb, torch_cuda, T, D, page, Hq, Hkv, prefix, lens, qlens):
    """With a table for 100,000 keys: the prefix in a pass of its own, or by every sequence's tiles."""
    c = Cache(torch_cuda, T, Hkv, D, page, lens, prefix=prefix, seed=prefix, width_more=100000 // page)
    p = lvb.attention_paged_plan(len(lens), Hq, Hkv, sum(qlens) + 3, max(qlens), page, c.table.shape[1], D=D,
                                 prefix_len=prefix)
    assert (p.kernel == lvb.PAGED_DECODE) <= (p.prefix_splits > 0)
    run_attention(lvb, torch_cuda, c, Hq, qlens, spare_rows=3)


@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("page,Hq,Hkv,prefix,lens,qlens,splits", [
    (16, 64, 8, 2003, [33, 0, 200, 3, 129] * 4, [3, 1, 2, 0, 3] * 4, 1),
    (64, 24, 8, 8193, [1500, 60, 7] * 3, [9, 1, 7] * 3, 2),       # own keys in ranges too
    (32, 6, 1, 20000, [30, 0, 2] * 20, [20, 3, 3] * 20, 1),       # rows of several tile pairs
    (32, 20, 4, 6000, [0] * 30, [5] * 30, 1),                     # no own keys at all
])
def test_shared_prefix_gathered(lvb, torch_cuda, T, D, page, Hq, Hkv, prefix, lens, qlens, splits):
    """More rows than the decoding kernel takes: the prefix read once for the rows of all sequences,
    and joined with the flash kernel's parts over their own keys."""
    c = Cache(torch_cuda, T, Hkv, D, page, lens, prefix=prefix, seed=prefix)
    p = lvb.attention_paged_plan(len(lens), Hq, Hkv, sum(qlens) + 3, max(qlens), page, c.table.shape[1], D=D,
                                 prefix_len=prefix)
    assert p.kernel == lvb.PAGED_FLASH and p.prefix_splits > 0 and p.launches == 3
    assert (p.splits > 1) == (splits > 1)
    run_attention(lvb, torch_cuda, c, Hq, qlens, spare_rows=3)
    run_attention(lvb, torch_cuda, c, Hq, qlens, causal=False)


@pytest.mark.parametrize("Hq,lens,qlens,prefix", [(8, [3000, 700, 5], [1, 1, 1], 0),
                                                  (8, [900, 333], [200, 333], 0),
                                                  (8, [100, 300], [1, 1], 2000)])
def test_large_scores(lvb, torch_cuda, Hq, lens, qlens, prefix):
    """Scores of several hundred: the reference maximum moves often and far."""
    c = Cache(torch_cuda, "fp16", 2, 128, 32, lens, prefix=prefix, seed=8)
    run_attention(lvb, torch_cuda, c, Hq, qlens, scale=20 * 128 ** -0.5)


@pytest.mark.parametrize("qlens", [[1, 1], [70, 33]])
def test_strides_and_uniform_rows(lvb, torch_cuda, qlens):
    """A cache with the heads before the slots, queries inside a fused projection, and (equal
    lengths) the call without cu_q."""
    torch = torch_cuda
    c = Cache(torch, "bf16", 2, 128, 16, [200, 77], seed=5, head_major=True)
    T = sum(qlens)
    qkv = torch.randn(T, 12, 128, device="cuda", generator=c.g).to(torch.bfloat16)
    run_attention(lvb, torch, c, 8, qlens, Q=qkv[:, 2:10])
    if qlens[0] == qlens[1]:
        run_attention(lvb, torch, c, 8, qlens, cu=False)
    # a bound on the rows that is above what any sequence has
    run_attention(lvb, torch, c, 8, qlens, max_q=qlens[0] + 2)


def test_many_sequences(lvb, torch_cuda):
    """More sequences than a CTA has threads, most of them idle."""
    rng = np.random.default_rng(1)
    lens = [int(x) if x > 40 else 0 for x in rng.integers(0, 400, 500)]
    qlens = [1 if n or i % 3 else 0 for i, n in enumerate(lens)]
    c = Cache(torch_cuda, "fp16", 1, 64, 16, lens, seed=9)
    run_attention(lvb, torch_cuda, c, 2, qlens)


def test_repeatable(lvb, torch_cuda):
    torch = torch_cuda
    for qlens, prefix in ([1] * 9, 0), ([1] * 9, 700), ([1] * 9, 9000), ([40] * 9, 0), ([9] * 9, 6000):
        c = Cache(torch, "bf16", 2, 128, 32, [2000, 3, 900, 50, 128, 4000, 77, 1, 600], prefix=prefix, seed=3)
        if qlens[0] > 1:
            c.seq_lens = c.seq_lens.clamp(min=0)
        Q = torch.randn(sum(qlens), 8, 128, device="cuda").to(torch.bfloat16)
        outs = []
        for _ in range(3):
            O = torch.empty_like(Q)
            lvb.attention_paged(O, Q, c.Kc, c.Vc, c.table, c.seq_lens, cu_q=cu_of(torch, qlens),
                                max_q=max(qlens),
                                **(dict(prefix_table=c.prefix_table, prefix_len=prefix) if prefix else {}))
            outs.append(O)
        torch.cuda.synchronize()
        status_ok(lvb)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- append -----------------------------------------------------------------------------------
@pytest.mark.parametrize("T,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("page,Hq,Hkv,lens,qlens,pairs,sections,layout,prefix", [
    (16, 8, 2, [1], [1], 32, None, "halves", 0),
    (8, 4, 4, [300, 5, 77, 16], [300, 1, 20, 0], 16, None, "pairs", 0),
    (48, 6, 1, [100, 60], [60, 60], 24, (8, 8, 8), "halves", 0),
    (64, 0, 3, [65, 64], [2, 1], 0, None, "halves", 0),           # no rotation, no queries
    (64, 0, 3, [65, 64], [2, 1], 32, None, "pairs", 1000),        # keys only, behind a prefix
    (32, 64, 8, [33] * 70, [1] * 70, 32, None, "halves", 0),
    (16, 2, 1, [20, 3, 9, 50, 1] * 300, [1, 0, 3, 0, 1] * 300, 32, None, "halves", 0),   # 1,500 entries
    (16, 2, 1, [0] * 700 + [70, 900] + [4] * 800, [0] * 700 + [70, 600] + [0] * 800, 16, None, "pairs", 0),
])
def test_append(lvb, torch_cuda, T, D, page, Hq, Hkv, lens, qlens, pairs, sections, layout, prefix):
    torch = torch_cuda
    c = Cache(torch, T, Hkv, D, page, lens, seed=page)
    Kc0, Vc0 = c.Kc.clone(), c.Vc.clone()
    n, spare = sum(qlens), 2
    dt = tdt(torch, T)
    K, V = (torch.randn(n + spare, Hkv, D, device="cuda", generator=c.g).to(dt) for _ in "kv")
    Q = torch.randn(n + spare, Hq, D, device="cuda", generator=c.g).to(dt) if Hq else None
    Qo = torch.full_like(Q, 7.0) if Hq else None
    axes = len(sections) if sections else 1
    place = np.concatenate([np.arange(a - q, a) for a, q in zip(lens, qlens)])
    pos = None
    if axes > 1:
        pos = torch.randint(0, 100000, (axes, n + spare), device="cuda", dtype=torch.int32, generator=c.g)
    f = freqs_of(torch, pairs) if pairs else None
    lvb.kv_append(c.Kc, c.Vc, K, V, c.table, c.seq_lens, cu_q=cu_of(torch, qlens), max_q=max(qlens),
                  Q=Q, Qo=Qo, pos=pos, freqs=f, sections=sections, layout=layout, prefix_len=prefix)
    torch.cuda.synchronize()
    status_ok(lvb)
    b = np.repeat(np.arange(len(lens)), qlens)
    pages = c.table.cpu().numpy()[b, place // page]
    pn = pos[:, :n].cpu().numpy() if pos is not None else (place + prefix)[None]
    assert torch.equal(c.Vc[pages, place % page], V[:n])
    got = c.Kc[pages, place % page]
    if pairs:
        ref = rotate(np64(K[:n]), pn[:, :, None], f.cpu().numpy(), list(sections) if sections else None, layout)
        assert (np.abs(np64(got) - ref) <= rot_bound(K[:n], ref, pairs, layout, T)).all()
    else:
        assert torch.equal(got, K[:n])
    if Hq:
        ref = rotate(np64(Q[:n]), pn[:, :, None], f.cpu().numpy(), list(sections) if sections else None, layout)
        assert (np.abs(np64(Qo[:n]) - ref) <= rot_bound(Q[:n], ref, pairs, layout, T)).all()
        assert bool((Qo[n:] == 7).all())
    # every other place is as it was (bit for bit: NaN among them)
    Kc0[pages, place % page] = got
    Vc0[pages, place % page] = V[:n]
    assert torch.equal(c.Kc.contiguous().view(torch.int16), Kc0.contiguous().view(torch.int16))
    assert torch.equal(c.Vc.contiguous().view(torch.int16), Vc0.contiguous().view(torch.int16))


def test_append_idle_entries_and_in_place(lvb, torch_cuda):
    """A padded decoding batch: entries of length 0 with a row each are left out; Q in place."""
    torch = torch_cuda
    c = Cache(torch, "bf16", 2, 128, 16, [5, 0, 33, 0], seed=2)
    before = c.Kc.clone()
    K, V, Q = (torch.randn(4, h, 128, device="cuda", generator=c.g).to(torch.bfloat16) for h in (2, 2, 4))
    Q0 = Q.clone()
    f = freqs_of(torch, 64)
    lvb.kv_append(c.Kc, c.Vc, K, V, c.table, c.seq_lens, Q=Q, Qo=Q, freqs=f)
    torch.cuda.synchronize()
    status_ok(lvb)
    assert torch.equal(Q[[1, 3]], Q0[[1, 3]])
    ref = rotate(np64(Q0[[0, 2]]), np.array([[4, 32]])[:, :, None], f.cpu().numpy())
    assert (np.abs(np64(Q[[0, 2]]) - ref) <= rot_bound(Q0[[0, 2]], ref, 64, "halves", "bf16")).all()
    changed = (c.Kc.view(torch.int16) != before.view(torch.int16)).flatten(1).any(1).nonzero().flatten()
    assert set(changed.tolist()) == {int(c.table[0, 0]), int(c.table[2, 2])}


def _step(lvb, torch, c, K, V, Q, qlens, lens, f, O, scale=None):
    """Append the new rows, then attend: lens counts them."""
    c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    cu = cu_of(torch, qlens)
    Qr = torch.empty_like(Q)
    lvb.kv_append(c.Kc, c.Vc, K, V, c.table, c.seq_lens, cu_q=cu, max_q=max(qlens), Q=Q, Qo=Qr, freqs=f)
    lvb.attention_paged(O, Qr, c.Kc, c.Vc, c.table, c.seq_lens, cu_q=cu, max_q=max(qlens))


def test_generation_equals_dense(lvb, torch_cuda):
    """Prompts in chunks and then token by token through append and paged attention, against the
    dense path (lvb.rope and lvb.attention) over the whole sequence: the two round K, P and O
    alike, but sum in another order, so they agree within twice the attention bound."""
    torch = torch_cuda
    B, Hq, Hkv, D, S, page = 3, 8, 2, 128, 75, 16
    g = torch.Generator(device="cuda").manual_seed(6)
    Q, K, V = (torch.randn(B, S, h, D, device="cuda", generator=g).to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    f = freqs_of(torch, 64)
    # dense: [B][H][S][D]
    Qd, Kd, Vd = (x.transpose(1, 2).contiguous() for x in (Q, K, V))
    pos = torch.arange(S, device="cuda", dtype=torch.int32)[None]
    lvb.rope(Qd, Qd, pos, f, Ko=Kd, K=Kd)
    Od = torch.empty_like(Qd)
    lvb.attention(Od, Qd, Kd, Vd, causal=True)
    # paged: chunks of uneven length, then single tokens; the pages are there from the start
    c = Cache(torch, "bf16", Hkv, D, page, [S] * B, seed=7)
    c.Kc.fill_(float("nan"))
    c.Vc.fill_(float("nan"))
    done = [0] * B
    O = torch.zeros(B, S, Hq, D, device="cuda", dtype=torch.bfloat16)
    for qlens in ([40, 1, 17], [20, 50, 17], [11, 20, 37], [1, 1, 1], [2, 2, 2], [1, 1, 1]):
        parts = [(b, slice(done[b], done[b] + q)) for b, q in enumerate(qlens)]
        cat = [torch.cat([x[b, s] for b, s in parts]) for x in (K, V, Q)]
        Os = torch.empty_like(cat[2])
        done = [d + q for d, q in zip(done, qlens)]
        _step(lvb, torch, c, *cat, qlens, done, f, Os)
        t = 0
        for (b, s), q in zip(parts, qlens):
            O[b, s] = Os[t:t + q]
            t += q
    torch.cuda.synchronize()
    status_ok(lvb)
    ref = Od.transpose(1, 2)
    mv = float(V.float().abs().max())
    for b in range(B):
        d = (O[b, :done[b]].double() - ref[b, :done[b]].double()).abs()
        assert bool((d <= 2 * (U["bf16"] * (mv + ref[b, :done[b]].double().abs()) + 2.0 ** -14 * mv)).all())


def test_captured_step_sees_new_lengths(lvb, torch_cuda):
    """Append and attention captured into two CUDA graphs, replayed while lengths, tokens and the
    table change, against the definition; eager calls run between the replays."""
    torch = torch_cuda
    c = Cache(torch, "fp16", 2, 64, 16, [100, 40, 64], seed=4)
    f = freqs_of(torch, 32)
    new = {k: torch.empty(3, h, 64, device="cuda", dtype=torch.float16) for k, h in (("K", 2), ("V", 2), ("Q", 4))}
    Qr, O = torch.empty_like(new["Q"]), torch.empty_like(new["Q"])
    lse = torch.empty(3, 4, device="cuda")
    app = lvb.prepare_kv_append(c.Kc, c.Vc, new["K"], new["V"], c.table, c.seq_lens, Q=new["Q"], Qo=Qr, freqs=f)
    att = lvb.prepare_attention_paged(O, Qr, c.Kc, c.Vc, c.table, c.seq_lens, lse=lse)
    for x in new.values():
        x.normal_(generator=c.g)
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        app()
        att()
        side.synchronize()
        for call in (app, att):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                call()
            graphs.append(graph)
    torch.cuda.synchronize()
    for step, lens in enumerate(([100, 40, 64], [101, 41, 65], [102, 1, 66], [103, 2, 0])):
        for b in range(3):          # pages for one more token
            if lens[b] and -(-lens[b] // 16) > int((c.table[b] >= 0).sum()):
                c.table[b, -(-lens[b] // 16) - 1] = c.spare.pop()
        for x in new.values():
            x.normal_(generator=c.g)
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        status_ok(lvb)
        eager, elser = torch.empty_like(O), torch.empty_like(lse)
        lvb.attention_paged(eager, Qr, c.Kc, c.Vc, c.table, c.seq_lens, lse=elser)
        torch.cuda.synchronize()
        assert torch.equal(eager, O) and torch.equal(elser, lse)
        for b, n in enumerate(lens):
            if n == 0:
                assert bool((O[b] == 0).all()) and bool(torch.isneginf(lse[b]).all())
                continue
            p = np.arange(n)
            pages = c.table.cpu().numpy()[b, p // 16]
            K, V = np64(c.Kc[pages, p % 16]), np64(c.Vc[pages, p % 16])
            ref = rotate(np64(new["K"][b]), np.array([[n - 1]]), f.cpu().numpy())
            assert np.abs(K[-1] - ref).max() <= 2.0 ** -9
            for h in range(2):
                o, l = attention_one(np64(Qr[b:b + 1, 2 * h:2 * h + 2]), K[:, h], V[:, h], n, 1, 0, True, 0.125)
                mv = np.abs(V[:, h]).max()
                assert (np.abs(np64(O[b:b + 1, 2 * h:2 * h + 2]) - o) <= U["fp16"] * (mv + np.abs(o)) + 2.0 ** -14 * mv).all()


def test_two_streams_at_once(lvb, torch_cuda):
    """The same call and others on two streams side by side: workspaces are each call's own."""
    torch = torch_cuda
    cs = [Cache(torch, "bf16", 4, 128, 64, [5000, 900, 3000], prefix=p, seed=s) for s, p in ((1, 0), (2, 600))]
    qs = [torch.randn(3, 32, 128, device="cuda").to(torch.bfloat16) for _ in cs]
    outs = [[torch.empty_like(q) for _ in range(6)] for q in qs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for i in range(6):
        for c, q, o, s in zip(cs, qs, outs, streams):
            more = dict(prefix_table=c.prefix_table, prefix_len=c.prefix) if c.prefix else {}
            lvb.attention_paged(o[i], q, c.Kc, c.Vc, c.table, c.seq_lens, stream=s, **more)
    torch.cuda.synchronize()
    status_ok(lvb)
    for o in outs:
        assert all(torch.equal(o[0], x) for x in o[1:]) and bool(torch.isfinite(o[0].float()).all())


def test_cache_beyond_32_bits(lvb, torch_cuda):
    """A cache of more than 2^32 bytes and 2^31 elements per tensor: the last pages."""
    torch = torch_cuda
    Hkv, D, page = 8, 128, 64
    pages = 2 ** 31 // (Hkv * D * page) + 50
    Kc = torch.zeros(pages, page, Hkv, D, device="cuda", dtype=torch.bfloat16)
    Vc = torch.zeros_like(Kc)
    assert Kc.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 200
    K, V = (torch.randn(n, Hkv, D, device="cuda", generator=g).to(torch.bfloat16) for _ in "kv")
    Q = torch.randn(n, 16, D, device="cuda", generator=g).to(torch.bfloat16)
    table = torch.tensor([[pages - 1, pages - 3, 0, pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    lvb.kv_append(Kc, Vc, K, V, table, lens)
    place = torch.arange(n, device="cuda")
    where = table[0].long()[place // page]
    assert torch.equal(Kc[where, place % page], K) and torch.equal(Vc[where, place % page], V)
    for rows in (1, n):
        O = torch.empty(rows, 16, D, device="cuda", dtype=torch.bfloat16)
        lvb.attention_paged(O, Q[n - rows:], Kc, Vc, table, lens)
        torch.cuda.synchronize()
        status_ok(lvb)
        for h in (0, 7):
            o, _ = attention_one(np64(Q[n - rows:, 2 * h:2 * h + 2]), np64(K[:, h]), np64(V[:, h]), n, rows, 0, True, D ** -0.5)
            mv = float(V.float().abs().max())
            assert (np.abs(np64(O[:, 2 * h:2 * h + 2]) - o) <= U["bf16"] * (mv + np.abs(o)) + 2.0 ** -14 * mv).all()


# ---- what the lists get wrong, found by the kernels' own checks -------------------------------
def test_bad_lists_are_reported(lvb, torch_cuda):
    """A length beyond the table, a page outside the cache and rows that do not fit: the status
    word names each, nothing outside the call's own rows and pages is written, and the sequences
    beside them are right."""
    torch = torch_cuda
    c = Cache(torch, "bf16", 2, 128, 16, [40, 70, 100], seed=6, width_more=0)
    Q = torch.randn(3, 4, 128, device="cuda").to(torch.bfloat16)
    good = torch.empty_like(Q)
    lvb.attention_paged(good, Q, c.Kc, c.Vc, c.table, c.seq_lens)
    status_ok(lvb)
    for lens, site in (([40, -1, 100], 81), ([40, 16 * 7 + 1, 100], 81)):
        O = torch.full_like(Q, 7.0)
        lvb.attention_paged(O, Q, c.Kc, c.Vc, c.table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
        code, where, _ = lvb.device_status()
        assert (code, where) == (lvb.LVB_ERR_INVALID_ARG, site)
        assert torch.equal(O[[0, 2]], good[[0, 2]]) and bool((O[1] == 0).all())
    for bad in (-1, c.Kc.shape[0], 2 ** 31 - 1):
        table = c.table.clone()
        table[1, 0] = bad
        O = torch.full_like(Q, 7.0)
        lvb.attention_paged(O, Q, c.Kc, c.Vc, table, c.seq_lens)
        code, where, _ = lvb.device_status()
        assert (code, where) == (lvb.LVB_ERR_INVALID_ARG, 82)
        assert torch.equal(O[[0, 2]], good[[0, 2]]) and bool(torch.isfinite(O[1].float()).all())
        before = (c.Kc.clone(), c.Vc.clone())
        last = table.clone()
        last[1, 4] = bad
        new = torch.randn(3, 2, 128, device="cuda").to(torch.bfloat16)
        lvb.kv_append(c.Kc, c.Vc, new, new, last, c.seq_lens)
        code, where, _ = lvb.device_status()
        assert (code, where) == (lvb.LVB_ERR_INVALID_ARG, 82)
        for b, n in ((0, 40), (2, 100)):
            before[0][int(table[b, (n - 1) // 16]), (n - 1) % 16] = new[b]
            before[1][int(table[b, (n - 1) // 16]), (n - 1) % 16] = new[b]
        assert torch.equal(c.Kc.view(torch.int16), before[0].view(torch.int16))
        assert torch.equal(c.Vc.view(torch.int16), before[1].view(torch.int16))
        lvb.attention_paged(good, Q, c.Kc, c.Vc, c.table, c.seq_lens)
        status_ok(lvb)
    for cu in ([0, 2, 1, 3], [0, 1, 3, 4], [-1, 0, 1, 2]):
        O = torch.full_like(Q, 7.0)
        lvb.attention_paged(O, Q, c.Kc, c.Vc, c.table, c.seq_lens,
                            cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=1)
        code, where, _ = lvb.device_status()
        assert (code, where) == (lvb.LVB_ERR_INVALID_ARG, 83)
    status_ok(lvb)
