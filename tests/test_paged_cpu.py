"""CPU tier: what the rotation, the paged cache's append and the paged attention refuse, how a
call is planned, and that their C structures match the ctypes ones. No GPU."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


def test_struct_layouts(lvb, tmp_path):
    structs = {"lvb_rotation": lvb.lvb_rotation, "lvb_rope_desc": lvb.lvb_rope_desc,
               "lvb_paged_desc": lvb.lvb_paged_desc, "lvb_append_desc": lvb.lvb_append_desc,
               "lvb_paged_plan": lvb.lvb_paged_plan}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "lvb.h"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    out = dict(l.rsplit(" ", 1) for l in subprocess.run(
        [str(exe)], capture_output=True, text=True, check=True).stdout.split("\n") if l)
    for name, cls in structs.items():
        assert int(out[name]) == C.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(out[f"{name}.{f}"]) == getattr(cls, f).offset, f"{name}.{f}"


def paged(lvb, **kw):
    d = lvb.lvb_paged_desc()
    d.dtype, d.causal = lvb.BF16, 1
    d.batch, d.heads_q, d.heads_kv, d.head_dim = 4, 8, 2, 128
    d.tokens, d.max_q, d.page_size, d.num_pages, d.table_width = 4, 1, 16, 100, 10
    d.scale = 0.1
    for k, v in kw.items():
        if isinstance(v, (list, tuple)):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


BAD_PAGED = [
    (dict(batch=-1), 1, "negative"),
    (dict(dtype=2), 2, "no kernel"),
    (dict(heads_kv=3), 1, "multiple of heads_kv"),
    (dict(heads_kv=0), 1, "multiple of heads_kv"),
    (dict(head_dim=96), 2, "head_dim"),
    (dict(page_size=0), 2, "page_size"),
    (dict(page_size=12), 2, "page_size"),
    (dict(num_pages=0), 1, "no page"),
    (dict(table_stride=9), 1, "table_stride"),
    (dict(table_width=2 ** 27), 2, "2^30"),
    (dict(prefix_len=2 ** 31), 2, "2^30"),
    (dict(num_pages=2 ** 31), 2, "2^31"),
    (dict(tokens=2 ** 31), 2, "2^31"),
    (dict(kc_stride=[4096, 256, 64]), 1, "K cache: stride"),
    (dict(vc_stride=[4096, 260, 128]), 2, "V cache: strides"),
    (dict(q_stride=[1024, 100]), 1, "Q: stride"),
    (dict(o_stride=[1028, 128]), 2, "result: strides"),
]


@pytest.mark.parametrize("kw,status,needle", BAD_PAGED + [
    (dict(scale=0.0), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"),
    (dict(heads_q=258), 2, "128 query heads"),
])
def test_attention_refusals(lvb, kw, status, needle):
    d = paged(lvb)
    assert lvb.lib.lvb_attention_paged_check(C.byref(d)) == 0
    d = paged(lvb, **kw)
    assert lvb.lib.lvb_attention_paged_check(C.byref(d)) == status
    msg = lvb.lib.lvb_last_error().decode()
    assert needle in msg and msg.startswith("lvb_attention_paged: ")


def append(lvb, rot=(64, 0, 1, 0, (64,)), **kw):
    d = lvb.lvb_append_desc()
    own = {k: kw.pop(k) for k in ("k_stride", "v_stride") if k in kw}
    d.paged = paged(lvb, **kw)
    for k, v in own.items():
        getattr(d, k)[:] = v
    d.rot.pairs, d.rot.layout, d.rot.n_axes, d.rot.inverse = rot[:4]
    d.rot.sections[:] = list(rot[4]) + [0] * (4 - len(rot[4]))
    return d


BAD_ROT = [((4, 0, 1, 0, (4,)), 2, "multiple of 8"), ((72, 0, 1, 0, (72,)), 2, "head_dim / 2"),
           ((-8, 0, 1, 0, (-8,)), 2, "multiple of 8"), ((64, 2, 1, 0, (64,)), 1, "layout"),
           ((64, 0, 0, 0, (64,)), 1, "n_axes"), ((64, 0, 5, 0, (64,)), 1, "n_axes"),
           ((64, 0, 2, 0, (32, 16)), 1, "add up"), ((64, 0, 2, 0, (72, -8)), 1, "negative section")]


@pytest.mark.parametrize("kw,status,needle", BAD_PAGED + [
    (dict(k_stride=[256, 120]), 1, "K: stride"),
    (dict(v_stride=[260, 128]), 2, "V: strides"),
] + [(dict(rot=r), s, n) for r, s, n in BAD_ROT])
def test_append_refusals(lvb, kw, status, needle):
    d = append(lvb)
    assert lvb.lib.lvb_kv_append_check(C.byref(d)) == 0
    d = append(lvb, **kw)
    assert lvb.lib.lvb_kv_append_check(C.byref(d)) == status
    msg = lvb.lib.lvb_last_error().decode()
    assert needle in msg and msg.startswith("lvb_kv_append: ")


def rope_desc(lvb, rot=(64, 0, 1, 0, (64,)), **kw):
    d = lvb.lvb_rope_desc()
    d.dtype, d.batch, d.heads_q, d.heads_kv, d.seq, d.head_dim = lvb.F32, 2, 4, 2, 10, 128
    for k, v in kw.items():
        if isinstance(v, (list, tuple)):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    d.rot.pairs, d.rot.layout, d.rot.n_axes, d.rot.inverse = rot[:4]
    d.rot.sections[:] = list(rot[4]) + [0] * (4 - len(rot[4]))
    return d


@pytest.mark.parametrize("kw,status,needle", [
    (dict(seq=-1), 1, "negative"),
    (dict(dtype=3), 2, "no kernel"),
    (dict(head_dim=40), 2, "head_dim"),
    (dict(head_dim=528), 2, "head_dim"),
    (dict(batch=70000), 2, "65535"),
    (dict(seq=2 ** 31), 2, "2^31"),
    (dict(q_stride=[5120, 1280, 64]), 1, "Q: stride"),
    (dict(ko_stride=[5120, 1282, 128]), 2, "rotated K: strides"),
    (dict(rot=(0, 0, 1, 0, (0,))), 1, "at least 8"),
] + [(dict(rot=r), s, n) for r, s, n in BAD_ROT])
def test_rope_refusals(lvb, kw, status, needle):
    d = rope_desc(lvb)
    assert lvb.lib.lvb_rope_check(C.byref(d)) == 0
    d = rope_desc(lvb, **kw)
    assert lvb.lib.lvb_rope_check(C.byref(d)) == status
    msg = lvb.lib.lvb_last_error().decode()
    assert needle in msg and msg.startswith("lvb_rope: ")


def test_calls_refuse_before_the_device(lvb):
    """NULL and misaligned pointers, rows without cu_q, a prefix without its table: found on the
    host; empty calls do nothing, without a device too."""
    lib, att = lvb.lib, lvb.lib.lvb_attention_paged
    d = paged(lvb)
    ok = [4096] * 7 + [4096, 4096, None]      # Q Kc Vc table lens cu prefix O lse stream

    def call(d, **at):
        a = list(ok)
        for i, v in at.items():
            a[int(i[1:])] = v
        return att(C.byref(d), *a), lib.lvb_last_error().decode()
    for i in (0, 1, 2, 7):
        assert call(d, **{f"p{i}": None})[0] == lvb.LVB_ERR_INVALID_ARG
        st, msg = call(d, **{f"p{i}": 4104})
        assert st == lvb.LVB_ERR_UNSUPPORTED and "16-byte" in msg
    for i in (3, 4):
        assert call(d, **{f"p{i}": None})[0] == lvb.LVB_ERR_INVALID_ARG
    for i in (3, 4, 5, 8):
        st, msg = call(d, **{f"p{i}": 4098})
        assert st == lvb.LVB_ERR_INVALID_ARG and "aligned" in msg
    st, msg = call(paged(lvb, tokens=5), p5=None)
    assert st == lvb.LVB_ERR_INVALID_ARG and "without cu_q" in msg
    st, msg = call(paged(lvb, prefix_len=3), p6=None)
    assert st == lvb.LVB_ERR_INVALID_ARG and "prefix_table" in msg
    assert att(None, *ok) == lvb.LVB_ERR_INVALID_ARG
    for empty in (dict(batch=0, tokens=0), dict(tokens=0), dict(max_q=0)):
        assert att(C.byref(paged(lvb, **empty)), *([None] * 10)) == 0

    app = lib.lvb_kv_append
    a = append(lvb)
    ok_a = [4096] * 11 + [None]               # Kc Vc K V Q Qo table lens cu pos freqs stream
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 10):
        args = list(ok_a)
        args[i] = None
        assert app(C.byref(a), *args) == lvb.LVB_ERR_INVALID_ARG, i
    none = append(lvb, rot=(0, 0, 1, 0, (0,)))
    assert app(C.byref(none), *ok_a) == lvb.LVB_ERR_INVALID_ARG      # Q without a rotation
    two = append(lvb, rot=(64, 0, 2, 0, (32, 32)))
    args = list(ok_a)
    args[9] = None
    assert app(C.byref(two), *args) == lvb.LVB_ERR_INVALID_ARG       # several axes without pos
    assert app(C.byref(append(lvb, tokens=0)), *([None] * 12)) == 0

    rope = lib.lvb_rope
    r = rope_desc(lvb)
    ok_r = [4096] * 6 + [None]                # Q K Qo Ko pos freqs stream
    for i in range(6):
        args = list(ok_r)
        args[i] = None
        assert rope(C.byref(r), *args) == lvb.LVB_ERR_INVALID_ARG, i
    args = list(ok_r)
    args[2] = 4104
    assert rope(C.byref(r), *args) == lvb.LVB_ERR_UNSUPPORTED
    assert rope(C.byref(rope_desc(lvb, seq=0)), *([None] * 7)) == 0


def test_python_refusals(lvb):
    import torch
    bf, i32 = torch.bfloat16, torch.int32
    Kc, Vc = torch.empty(10, 16, 2, 128, dtype=bf), torch.empty(10, 16, 2, 128, dtype=bf)
    Q, O = torch.empty(3, 8, 128, dtype=bf), torch.empty(3, 8, 128, dtype=bf)
    table, lens = torch.zeros(3, 4, dtype=i32), torch.zeros(3, dtype=i32)
    cu = torch.zeros(4, dtype=i32)
    att = dict(O=O, Q=Q, Kc=Kc, Vc=Vc, block_table=table, seq_lens=lens)

    def refused(f, needle, **kw):
        with pytest.raises(lvb.LavaError) as e:
            f(**kw)
        assert needle in str(e.value)
    for change, needle in [
            (dict(O=O[:2]), "Q and O"), (dict(Q=Q[..., :64], O=O[..., :64]), "Q and O"),
            (dict(Vc=Vc[:9]), "caches"), (dict(Vc=Vc.half()), "caches"),
            (dict(block_table=table.long()), "block_table"), (dict(block_table=table[0]), "block_table"),
            (dict(seq_lens=lens[:2]), "seq_lens"), (dict(seq_lens=lens.long()), "seq_lens"),
            (dict(cu_q=cu), "max_q"), (dict(cu_q=cu[:3], max_q=1), "cu_q"),
            (dict(block_table=table[:2], seq_lens=lens[:2]), "pass cu_q"),
            (dict(Q=Q.half(), O=O.half()), "dtype"),
            (dict(prefix_len=20), "prefix_table"),
            (dict(prefix_len=20, prefix_table=torch.zeros(1, dtype=i32)), "prefix_table has 1"),
            (dict(lse=torch.empty(3, 8, dtype=bf)), "lse"), (dict(lse=torch.empty(8, 3).t()), "lse"),
            (dict(Kc=Kc.transpose(0, 3).contiguous().transpose(0, 3)), "contiguous"),
            (dict(), "not a CUDA tensor")]:
        refused(lvb.attention_paged, needle, **{**att, **change})
    K, V = torch.empty(3, 2, 128, dtype=bf), torch.empty(3, 2, 128, dtype=bf)
    f = torch.ones(64, dtype=torch.float64)
    app = dict(Kc=Kc, Vc=Vc, K=K, V=V, block_table=table, seq_lens=lens)
    for change, needle in [
            (dict(Q=Q), "come together"), (dict(Q=Q, Qo=O), "without freqs"),
            (dict(pos=lens), "without freqs"), (dict(freqs=f.float()), "freqs"),
            (dict(freqs=f, layout="thirds"), "layout"), (dict(freqs=f, sections=(32, 32)), "need pos"),
            (dict(freqs=f, sections=(32, 16), pos=torch.zeros(2, 3, dtype=i32)), "add up"),
            (dict(freqs=f, pos=torch.zeros(4, dtype=i32)), "pos"),
            (dict(freqs=f, pos=torch.zeros(3)), "pos"),
            (dict(V=V[:2]), "V must be"), (dict(K=K.half()), "K must be"),
            (dict(freqs=f, Q=Q, Qo=O[:, :4]), "Qo must be"), (dict(freqs=f), "not a CUDA tensor")]:
        refused(lvb.kv_append, needle, **{**app, **change})
    X = torch.empty(2, 4, 5, 128)
    rp = dict(Qo=X, Q=X, pos=torch.zeros(2, 5, dtype=i32), freqs=f)
    for change, needle in [
            (dict(Qo=X[:1]), "one shape"), (dict(K=X), "come together"),
            (dict(K=X[:1], Ko=X[:1]), "K and Ko"), (dict(Qo=X.half()), "dtype"),
            (dict(pos=torch.zeros(3, 5, dtype=i32)), "pos"), (dict(pos=torch.zeros(2, 5)), "int32"),
            (dict(sections=(32, 32)), "pos"), (dict(freqs=f[:60]), "multiple of 8"),
            (dict(sections=(8,) * 5), "1 to 4"), (dict(), "not a CUDA tensor")]:
        refused(lvb.rope, needle, **{**rp, **change})


def test_plans(lvb):
    """Few rows per KV head take the decoding kernel, more the flash kernel, with its key range
    split when the tiles alone cannot fill the SMs; a prefix is read once for all by the decoding
    form and by every sequence's tiles in the other."""
    p = lvb.attention_paged_plan(8, 64, 8, 8, 1, 64, 256)
    assert (p.kernel, p.prefix_splits, p.launches) == (lvb.PAGED_DECODE, 0, 2)
    assert p.workspace_bytes == 64 * 16 + 2 * 148 * 16 * 130 * 4
    p = lvb.attention_paged_plan(8, 64, 8, 8, 1, 64, 256, prefix_len=16384)
    assert (p.kernel, p.prefix_splits, p.cluster, p.launches) == (lvb.PAGED_DECODE, 16, 0, 3)
    assert lvb.attention_paged_plan(64, 32, 8, 64, 1, 16, 4, prefix_len=500).prefix_splits > 0
    # ... and few or short sequences by the decoding form, each in front of its own keys
    for args, cluster in [((4, 32, 8, 4, 1, 16, 4), 3), ((32, 32, 8, 32, 1, 16, 4), 0)]:
        p = lvb.attention_paged_plan(*args, prefix_len=500)
        assert (p.kernel, p.prefix_splits, p.cluster, p.launches) == (lvb.PAGED_DECODE, 0, cluster, 1)
    # few or short sequences: clusters of CTAs, one launch, no workspace
    for args, cluster in [((1, 32, 8, 1, 1, 16, 49), 7), ((1, 32, 8, 1, 1, 16, 100), 7),
                          ((1, 32, 8, 1, 1, 16, 640), 10), ((1, 32, 8, 1, 1, 16, 641), 0),
                          ((1, 32, 8, 1, 1, 16, 1), 1), ((2, 32, 8, 2, 1, 16, 512), 0),
                          ((8, 32, 8, 8, 1, 16, 64), 2), ((16, 32, 8, 16, 1, 16, 64), 1),
                          ((32, 32, 8, 32, 1, 16, 72), 0)]:
        p = lvb.attention_paged_plan(*args)
        assert p.cluster == cluster, (args, p.cluster)
        assert (p.launches, p.workspace_bytes == 0) == ((1, True) if cluster else (2, False))
    # many short ones: whole items, the same
    p = lvb.attention_paged_plan(32, 32, 8, 32, 1, 16, 64)
    assert (p.cluster, p.launches, p.workspace_bytes) == (0, 1, 0)
    assert lvb.attention_paged_plan(8, 64, 8, 16, 2, 64, 256).kernel == lvb.PAGED_DECODE    # 16 rows
    assert lvb.attention_paged_plan(8, 64, 8, 24, 3, 64, 256).kernel == lvb.PAGED_FLASH     # 24 rows
    # ... behind a long prefix: its keys once for the rows of all sequences, then theirs beside them
    p = lvb.attention_paged_plan(32, 64, 8, 128, 4, 64, 5, prefix_len=16384)
    assert (p.kernel, p.splits, p.cluster, p.launches) == (lvb.PAGED_FLASH, 1, 0, 3)
    assert p.prefix_splits == 4
    parts = 4 * 8 * 4 * 256 * 130 * 4 + 256                       # four tile pairs, eight KV heads
    assert p.workspace_bytes == parts + 32 * 8 * 256 * 130 * 4 + 256
    p = lvb.attention_paged_plan(1, 32, 8, 64, 64, 64, 1000)
    assert (p.kernel, p.splits, p.cluster, p.launches) == (lvb.PAGED_FLASH, 18, 2, 2)
    p = lvb.attention_paged_plan(1, 32, 8, 64, 64, 64, 4)             # two blocks of keys
    assert (p.splits, p.cluster, p.launches) == (2, 2, 1)
    p = lvb.attention_paged_plan(1, 32, 8, 64, 64, 64, 2)             # one: no split
    assert (p.splits, p.cluster, p.launches) == (1, 0, 1)
    p = lvb.attention_paged_plan(16, 32, 8, 16384, 2048, 64, 1000, prefix_len=500)
    assert (p.kernel, p.splits, p.prefix_splits, p.launches) == (lvb.PAGED_FLASH, 1, 0, 1)
    assert lvb.attention_paged_plan(0, 32, 8, 0, 1, 64, 4).launches == 0
    # the join's rows are counted in 32 bits; parts beyond 512 MiB are not gathered
    with pytest.raises(lvb.LavaError, match="split the batch"):
        lvb.attention_paged_plan(2 ** 25 + 1, 16, 1, 2 ** 25 + 1, 1, 128, 16)
    assert lvb.attention_paged_plan(400, 64, 8, 1600, 4, 64, 5, prefix_len=16384).prefix_splits > 0
    assert lvb.attention_paged_plan(600, 64, 8, 2400, 4, 64, 5, prefix_len=16384).prefix_splits == 0
