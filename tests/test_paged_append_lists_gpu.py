"""GPU tier: kv_append with lists that are wrong, found by the kernel's own checks: whichever sequence they are
wrong for, also one without new rows, the status word names the site, nothing outside the tokens' own places
is written, and what is written is right."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Append:
    def __init__(self, lvb, torch, lens, qlens, page=16, Hq=4, Hkv=2, D=64, max_q=None):
        self.lvb, self.torch, self.page = lvb, torch, page
        g = torch.Generator(device="cuda").manual_seed(len(lens))
        counts = [-(-n // page) for n in lens]
        self.lens, self.max_q = list(lens), max_q or max(qlens)
        self.cu = [0] + [int(x) for x in np.cumsum(qlens)]
        self.tokens = self.cu[-1] + 2
        self.pages = sum(counts) + 3
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32)
        self.width = max(counts) + 1
        table = torch.full((len(lens), self.width), -7, dtype=torch.int32)
        at, order = 0, order.cpu()
        for b, n in enumerate(counts):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table.cuda()
        shape = (self.pages, page, Hkv, D)
        self.cache = [torch.randn(shape, device="cuda", generator=g).half() for _ in "kv"]
        self.K, self.V = (torch.randn(self.tokens, Hkv, D, device="cuda", generator=g).half() for _ in "kv")
        self.Q = torch.randn(self.tokens, Hq, D, device="cuda", generator=g).half()
        self.f = torch.exp(-torch.arange(D // 2, dtype=torch.float64, device="cuda") * 0.3)
        # positions of their own, so that a token's rotation does not depend on its sequence
        self.pos = torch.arange(self.tokens, device="cuda", dtype=torch.int32) * 3
        self.Kr, self.Qr = torch.empty_like(self.K), torch.empty_like(self.Q)
        lvb.rope(self.Qr.transpose(0, 1)[None], self.Q.transpose(0, 1)[None], self.pos[None], self.f,
                 Ko=self.Kr.transpose(0, 1)[None], K=self.K.transpose(0, 1)[None])

    def run(self, site, lens=None, cu=None, table=None, may_miss=False):
        torch, lvb = self.torch, self.lvb
        lens, cu = lens or self.lens, cu or self.cu
        table = self.table if table is None else table
        Kc, Vc = (x.clone() for x in self.cache)
        Qo = torch.full_like(self.Q, 7.0)
        ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, cu)]
        lvb.kv_append(Kc, Vc, self.K, self.V, table, ints[0], cu_q=ints[1], max_q=self.max_q, Q=self.Q, Qo=Qo,
                      pos=self.pos, freqs=self.f)
        torch.cuda.synchronize()
        code, where, _ = lvb.device_status()
        assert (code, where) == ((lvb.LVB_ERR_INVALID_ARG, site) if site else (0, 0)), (lens, cu)
        # what the lists say of each token
        want = {}
        rows = table.cpu().numpy()
        for b, n in enumerate(lens):
            r0, r1 = cu[b], cu[b + 1]
            if not (0 <= r1 - r0 <= self.max_q and 0 <= r0 and r1 <= self.tokens):
                continue
            if not 0 <= n <= self.width * self.page:
                n = 0
            for t in range(r0, r1):
                place = n - (r1 - t)
                if place >= 0 and 0 <= rows[b, place // self.page] < self.pages:
                    want[t] = rows[b, place // self.page], place % self.page
        done = (Qo != 7).flatten(1).any(1).nonzero().flatten().tolist()
        if may_miss:
            assert set(done) <= set(want)
        else:
            assert done == sorted(want)
        K0, V0 = (x.clone() for x in self.cache)
        if done:
            page, slot = (torch.tensor([int(want[t][i]) for t in done], device="cuda") for i in (0, 1))
            K0[page, slot], V0[page, slot] = self.Kr[done], self.V[done]
            assert torch.equal(Qo[done], self.Qr[done])
        assert torch.equal(Kc, K0) and torch.equal(Vc, V0)
        return len(done)


@pytest.mark.parametrize("lens,qlens", [
    ([40, 70, 100], [1, 1, 1]),
    ([40, 0, 100, 33], [3, 0, 20, 1]),
    ([16, 3, 9, 50, 1] * 20, [1, 0, 3, 4, 1] * 20),
    ([9, 17] * 700, [1, 2] * 700),                        # more than one round of the search
])
def test_wrong_lists(lvb, torch_cuda, lens, qlens):
    c = Append(lvb, torch_cuda, lens, qlens)
    assert c.run(None) == sum(qlens)
    B = len(lens)
    for b in {0, 1, B // 2, B - 1}:
        for n in (-1, -2 ** 31, c.width * c.page + 1, 2 ** 31 - 1):
            c.run(81, lens=lens[:b] + [n] + lens[b + 1:])              # (sequence 1 may have no rows)
    for page in (-1, c.pages, 2 ** 31 - 1):
        table = c.table.clone()
        b = int(np.argmax(qlens))
        table[b, (lens[b] - 1) // c.page] = page
        c.run(82, table=table)
    c.run(83, cu=c.cu[:-1] + [c.tokens + 1])
    c.run(83, cu=c.cu[:-1] + [2 ** 31 - 1])
    # rows before the first, fewer than none, a list out of order: tokens beside it may be missed, none
    # goes anywhere else
    for b in {0, B // 2, B - 1}:
        for x in (-1, -2 ** 31, c.cu[b + 1] + 1, 2 ** 31 - 1):
            if b and 0 <= x - c.cu[b - 1] <= c.max_q and b < B - 1:
                continue                    # the sequence before it would share rows with the one behind it
            c.run(83, cu=c.cu[:b] + [x] + c.cu[b + 1:], may_miss=True)
    assert c.run(None) == sum(qlens)


def test_more_rows_than_announced(lvb, torch_cuda):
    c = Append(lvb, torch_cuda, [40, 70, 100], [2, 5, 1], max_q=4)
    assert c.run(83) == 3


def test_idle_sequences_are_no_fault(lvb, torch_cuda):
    """Entries without rows and without keys among the others, and rows behind the last sequence."""
    c = Append(lvb, torch_cuda, [0, 40, 0, 0, 17, 0], [0, 2, 0, 0, 1, 0])
    assert c.run(None) == 3
