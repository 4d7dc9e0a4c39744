"""CPU tier: tensors whose elements several rows share (torch's expand) are refused where the C
interface would take their zero strides for a packed layout and address rows that are not there.
Nothing here runs a kernel: the refusals come before the device is looked for."""
import pytest
import torch

BF, I32 = torch.bfloat16, torch.int32


def wide(*shape, dtype=BF):
    """One head's elements under every row of `shape`: strides (0, ..., 0, 1)."""
    t = torch.zeros(shape[-1], dtype=dtype).expand(*shape)
    assert all(s == 0 for s in t.stride()[:-1])
    return t


def refused(lvb, f, args, change, name):
    with pytest.raises(lvb.LavaError) as e:
        f(**{**args, **change})
    assert "not a CUDA tensor" not in str(e.value)
    assert f"{name}: stride below head_dim" in str(e.value)


def same(args, op, lvb):
    """The unchanged call gets as far as the look for the device."""
    with pytest.raises(lvb.LavaError, match="not a CUDA tensor"):
        op(**args)


@pytest.mark.parametrize("name", ["Q", "Qo", "K", "Ko"])
def test_rope_refuses_expanded(lvb, name):
    X = {n: torch.empty(2, 3, 5, 128) for n in ("Q", "Qo", "K", "Ko")}
    args = dict(**X, pos=torch.zeros(2, 5, dtype=I32), freqs=torch.ones(64, dtype=torch.float64))
    same(args, lvb.rope, lvb)
    refused(lvb, lvb.rope, args, {name: wide(2, 3, 5, 128, dtype=torch.float32)}, name)
    # the gradient of a sum over heads: only some of the strides are 0
    some = torch.zeros(2, 1, 5, 128).expand(2, 3, 5, 128)
    refused(lvb, lvb.rope, args, {name: some, "inverse": True}, name)


@pytest.mark.parametrize("name,shape", [("Kc", (10, 16, 2, 128)), ("Vc", (10, 16, 2, 128)),
                                        ("K", (3, 2, 128)), ("V", (3, 2, 128)),
                                        ("Q", (3, 8, 128)), ("Qo", (3, 8, 128))])
def test_append_refuses_expanded(lvb, name, shape):
    c, n, q = (10, 16, 2, 128), (3, 2, 128), (3, 8, 128)
    args = {k: torch.empty(s, dtype=BF)
            for k, s in (("Kc", c), ("Vc", c), ("K", n), ("V", n), ("Q", q), ("Qo", q))}
    args.update(block_table=torch.zeros(3, 4, dtype=I32), seq_lens=torch.zeros(3, dtype=I32),
                freqs=torch.ones(64, dtype=torch.float64))
    same(args, lvb.kv_append, lvb)
    refused(lvb, lvb.kv_append, args, {name: wide(*shape)}, name)


@pytest.mark.parametrize("name,shape", [("Kc", (10, 16, 2, 128)), ("Vc", (10, 16, 2, 128)),
                                        ("Q", (3, 8, 128)), ("O", (3, 8, 128))])
def test_attention_refuses_expanded(lvb, name, shape):
    args = dict(O=torch.empty(3, 8, 128, dtype=BF), Q=torch.empty(3, 8, 128, dtype=BF),
                Kc=torch.empty(10, 16, 2, 128, dtype=BF), Vc=torch.empty(10, 16, 2, 128, dtype=BF),
                block_table=torch.zeros(3, 4, dtype=I32), seq_lens=torch.zeros(3, dtype=I32))
    same(args, lvb.attention_paged, lvb)
    refused(lvb, lvb.attention_paged, args, {name: wide(*shape)}, name)


def test_rows_of_extent_one_may_have_any_stride(lvb):
    """A dimension of one row has no stride that counts."""
    Q = torch.zeros(128, dtype=BF).as_strided((1, 1, 128), (0, 0, 1))
    args = dict(O=torch.empty(1, 1, 128, dtype=BF), Q=Q,
                Kc=torch.empty(1, 8, 1, 128, dtype=BF), Vc=torch.empty(1, 8, 1, 128, dtype=BF),
                block_table=torch.zeros(1, 1, dtype=I32), seq_lens=torch.zeros(1, dtype=I32))
    same(args, lvb.attention_paged, lvb)


@pytest.mark.parametrize("call", ["attention_paged", "kv_append"])
def test_expanded_table_is_refused(lvb, call):
    """One row of pages expanded over the sequences: a row stride of 0 stands for packed rows in the
    descriptor, so the entries behind the row would be read. Rows that overlap are refused too."""
    Kc, Vc = (torch.empty(10, 16, 2, 128, dtype=BF) for _ in "kv")
    X, Y = (torch.empty(3, 2, 128, dtype=BF) for _ in "xy")
    names = ("O", "Q") if call == "attention_paged" else ("K", "V")
    args = dict(zip(names, (X, Y)), Kc=Kc, Vc=Vc, seq_lens=torch.zeros(3, dtype=I32),
                block_table=torch.zeros(3, 4, dtype=I32))
    f = getattr(lvb, call)
    same(args, f, lvb)
    for table in (torch.zeros(1, 4, dtype=I32).expand(3, 4), torch.zeros(1, 1, dtype=I32).expand(3, 1),
                  torch.zeros(12, dtype=I32).as_strided((3, 4), (2, 1))):
        with pytest.raises(lvb.LavaError, match="block_table: stride below its width"):
            f(**{**args, "block_table": table})
    for table in (torch.zeros(3, 9, dtype=I32)[:, :4], torch.zeros(3, 0, dtype=I32)):
        same({**args, "block_table": table}, f, lvb)
    one = {k: v[:1] if k in names + ("seq_lens",) else v for k, v in args.items()}
    same({**one, "block_table": torch.zeros(4, dtype=I32).as_strided((1, 4), (0, 1))}, f, lvb)
