"""GPU tier: long flat tails of small weights. A few keys hold almost all the weight and thousands hold
2^-25.5 of it each: the sum of the many counts, in the result as in lse, whatever type the weights are
rounded to for the product with V.

Tolerance, per element, from the kernels' arithmetic (u = half a step of the type, 2^-8 bf16, 2^-11 fp16):
  u·(Σ p|V| + |O|)       each weight above the type's subnormals, and O at its store, rounded once
  2^-31·Σ|V| / Σ 2^(s-max)   fp16: weights that fall among its subnormals. They are held 2^6 above their
                         value (the reference maximum weighs 2^6, or up to 2^14 while it is let
                         stand), a step there is 2^-24 and a rounding half of it, 2^-25 · 2^-6; the
                         reference is at most the maximum, and a part's own is no larger
  2^-14·Σ p|V|           scores, exponentials and sums in 32 bits (as in tests/test_paged_gpu.py)
  2^-25                  fp16: half a step of O's own subnormals.
The scores are exact (one product of two values), all rows are alike, and V is positive, so a lost tail
shows as an error of the size of the result.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
HOT = 25.5 * np.log(2.0)


@pytest.mark.parametrize("T,D", [("fp16", 128), ("bf16", 128), ("fp16", 64), ("bf16", 64)])
@pytest.mark.parametrize("form,batch,Hq,Hkv,q,own,prefix,more", [
    ("flash, whole tiles", 10, 8, 8, 20, 4096, 0, 0),
    ("flash, ranges joined in clusters", 1, 4, 1, 9, 4096, 0, 0),
    ("flash, ranges joined from memory", 1, 32, 8, 64, 8192, 0, 100000),
    ("flash, the prefix in front", 10, 16, 8, 128, 512, 3000, 0),
    ("flash, the prefix gathered", 32, 64, 8, 4, 512, 8192, 0),
    ("decoding, the prefix gathered", 32, 32, 8, 1, 512, 8192, 100000),
    ("decoding, dealt", 3, 32, 8, 2, 4096, 0, 100000),
    ("decoding, clusters", 1, 8, 8, 1, 900, 0, 0),
])
def test_flat_tail(lvb, torch_cuda, T, D, form, batch, Hq, Hkv, q, own, prefix, more):
    torch = torch_cuda
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[T]
    page = 64
    g = torch.Generator(device="cuda").manual_seed(own + prefix)
    n = own + prefix
    K = torch.zeros(n, Hkv, D, device="cuda", dtype=dt)
    K[::512, :, 0] = HOT / 4
    V = (0.5 + torch.rand(n, Hkv, D, device="cuda", generator=g)).to(dt)
    V[::512] = 0
    pages = -(-own // page), -(-prefix // page)
    order = torch.randperm(sum(pages), device="cuda", generator=g).to(torch.int32)
    Kc, Vc = (torch.zeros(sum(pages), page, Hkv, D, device="cuda", dtype=dt) for _ in "kv")
    rows = order[:pages[0]], order[pages[0]:].contiguous()
    for row, part in ((rows[1], slice(0, prefix)), (rows[0], slice(prefix, n))):
        at = torch.arange(part.stop - part.start, device="cuda")
        Kc[row.long()[at // page], at % page] = K[part]
        Vc[row.long()[at // page], at % page] = V[part]
    # all sequences read the same pages
    table = torch.zeros(batch, pages[0] + more // page, device="cuda", dtype=torch.int32)
    table[:, :pages[0]] = rows[0]
    lens = torch.full((batch,), own, device="cuda", dtype=torch.int32)
    Q = torch.zeros(batch * q, Hq, D, device="cuda", dtype=dt)
    Q[..., 0] = 4
    O, lse = torch.empty_like(Q), torch.empty(batch * q, Hq, device="cuda")
    plan = lvb.attention_paged_plan(batch, Hq, Hkv, batch * q, q, page, table.shape[1], D=D, causal=False,
                                    prefix_len=prefix)
    assert (plan.kernel == lvb.PAGED_DECODE) == form.startswith("decoding"), form
    assert (plan.prefix_splits > 0) == form.endswith("gathered"), form
    assert plan.cluster > 1 or "clusters" not in form, form
    assert (plan.launches > 1) == ("memory" in form or "gathered" in form or "dealt" in form), form
    lvb.attention_paged(O, Q, Kc, Vc, table, lens, max_q=q, causal=False, scale=1.0, lse=lse,
                        **(dict(prefix_table=rows[1], prefix_len=prefix) if prefix else {}))
    torch.cuda.synchronize()
    assert lvb.device_status() == (0, 0, 0)
    s = 4.0 * K[:, :, 0].double()                                   # [key][KV head]
    w = torch.exp(s - s.amax(0))
    l = w.sum(0)
    ref = torch.einsum("nh,nhd->hd", w, V.double()) / l[:, None]     # also Σ p|V|
    lref = s.amax(0) + torch.log(l)
    bound = U[T] * 2 * ref + 2.0 ** -14 * ref
    if T == "fp16":
        bound = bound + 2.0 ** -31 * V.double().sum(0) / l[:, None] + 2.0 ** -25
    got = O.view(-1, Hkv, Hq // Hkv, D).double()
    err = (got - ref[None, :, None]).abs()
    assert bool((err <= bound[None, :, None]).all()), (float(err.max()), float(bound.max()), float(ref.min()))
    lerr = (lse.view(-1, Hkv, Hq // Hkv).double() - lref[None, :, None]).abs()
    assert bool((lerr <= 2.0 ** -14 * (1 + lref.abs())[None, :, None]).all())
