"""Arguments that the operators for several tokens a step refuse.  The C ABI checks them before any CUDA call, so that plain host
tensors show it; the calls that would be accepted are not made here."""

import pytest
import torch

from pariskv_b200 import _lib as L

BF, I32, U8 = torch.bfloat16, torch.int32, torch.uint8


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def call(name, args):
    keep = [L.desc(a) if isinstance(a, torch.Tensor) else a for a in args]
    rc = getattr(L.load(), name)(*[L.ref(a) if isinstance(a, L.PkTensor) else a for a in keep])
    return rc, L.load().pk_last_error().decode()


def refused(name, args, match, code=1):
    rc, msg = call(name, args)
    assert rc == code and match in msg, (rc, msg)


def odd(t):
    """The same shape, rows at a stride that is no multiple of 8."""
    return z(*t.shape[:-1], t.shape[-1] + 4)[..., :t.shape[-1]]


TREE = dict(q=z(2, 3, 4, 128), k=z(2, 2, 16, 128), v=z(2, 2, 16, 128), dk=z(2, 3, 2, 128), dv=z(2, 3, 2, 128), mask=z(2, 3, 3, dtype=U8),
            lengths=z(2, dtype=I32), scale=0.1, out=z(2, 3, 4, 128), lse=None, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(q=None), "queries is null"), (dict(q=z(2, 3, 4, 128, dtype=torch.float32)), "dtype"), (dict(q=z(2, 3, 4, 64)), "queries must be"),
    (dict(q=odd(TREE["q"])), "multiples of 8"), (dict(k=odd(TREE["k"])), "multiples of 8"), (dict(k=z(1, 2, 16, 128)), "keys must be"),
    (dict(v=z(2, 2, 15, 128)), "shape of keys"), (dict(q=z(2, 3, 3, 128)), "multiple of the KV heads"), (dict(lengths=z(3, dtype=I32)), "lengths must be"),
    (dict(lengths=z(4, dtype=I32)[::2]), "lengths must be"), (dict(out=z(2, 3, 4, 256)[..., ::2]), "out must be"), (dict(out=z(2, 3, 2, 128)), "shape of queries"),
    (dict(lse=z(2, 3, 2, dtype=torch.float32)), "lse must be"), (dict(dk=z(2, 4, 2, 128)), "draft_keys"), (dict(dv=odd(TREE["dv"])), "multiples of 8"),
    (dict(mask=z(3, 3, 3, dtype=U8)), "tree_mask must be"), (dict(mask=z(2, 3, 4, dtype=U8)), "tree_mask must be"), (dict(mask=z(2, 3, 3, dtype=I32)), "dtype"),
    (dict(q=z(1, 300, 4, 128), k=z(1, 2, 16, 128), v=z(1, 2, 16, 128), dk=z(1, 300, 2, 128), dv=z(1, 300, 2, 128), mask=z(1, 300, 300, dtype=U8),
          lengths=z(1, dtype=I32), out=z(1, 300, 4, 128)), "at most 256"), (dict(q=z(2, 3, 1032, 128), out=z(2, 3, 1032, 128)), "at most 128")])
def test_tree_attention(change, match):
    refused("pk_tree_attention", list({**TREE, **change}.values()), match)


BOUNDS = dict(k=z(2, 2, 40, 128), lengths=z(2, dtype=I32), block=16, n_new=-1, out=z(2, 2, 3, 2, 128), stream=None)


@pytest.mark.parametrize("change,match", [(dict(block=8), "block must be"), (dict(block=0), "block must be"), (dict(n_new=-2), "n_new"),
                                          (dict(out=z(2, 2, 2, 2, 128)), "bounds must be"), (dict(out=z(2, 2, 3, 128, 2).transpose(3, 4)), "bounds"),
                                          (dict(k=odd(BOUNDS["k"])), "multiples of 8"), (dict(lengths=z(1, dtype=I32)), "lengths must be"), (dict(k=z(2, 2, 40, 64)), "keys must be")])
def test_block_bounds(change, match):
    refused("pk_block_bounds", list({**BOUNDS, **change}.values()), match)


SELECT = dict(q=z(2, 1, 4, 128), bounds=z(2, 2, 3, 2, 128), lengths=z(2, dtype=I32), block=16, sink=1, local=1, blocks=z(2, 1, 2, 2, dtype=I32), ws=None,
              ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,match,code", [
    (dict(block=100), "block must be", 1), (dict(sink=2), "no more sink and local", 1), (dict(local=0), "at least one local", 1), (dict(sink=-1), "sink", 1),
    (dict(q=z(2, 1, 3, 128)), "multiple of the KV heads", 1), (dict(q=odd(SELECT["q"])), "multiples of 8", 1), (dict(blocks=z(2, 1, 1, 2, dtype=I32)), "blocks must be", 1),
    (dict(blocks=z(2, 1, 2, 2, dtype=torch.int64)), "dtype", 1), (dict(bounds=z(1, 2, 3, 2, 128)), "multiple of the KV heads", 1)])
def test_select_blocks(change, match, code):
    refused("pk_select_blocks", list({**SELECT, **change}.values()), match, code)


ATTEND = dict(q=z(2, 1, 4, 128), k=z(2, 2, 40, 128), v=z(2, 2, 40, 128), blocks=z(2, 1, 2, 2, dtype=I32), lengths=z(2, dtype=I32), block=16, scale=0.1,
              out=z(2, 1, 4, 128), lse=None, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,match", [(dict(block=48), "block must be"), (dict(blocks=z(2, 1, 2, 4, dtype=I32)[..., ::2]), "blocks must be"),
                                          (dict(blocks=z(2, 2, 2, 2, dtype=I32)), "blocks must be"), (dict(v=odd(ATTEND["v"])), "multiples of 8"), (dict(lengths=None), "lengths is null")])
def test_block_attention(change, match):
    refused("pk_block_attention", list({**ATTEND, **change}.values()), match)


W4 = dict(w=z(6, 64, dtype=U8), scales=z(6, 2), offsets=None, x=z(3, 128), out=z(3, 6), gated=0, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(scales=z(6, 8)), "group must be"), (dict(scales=z(6, 3)), "scales must be"), (dict(scales=z(5, 2)), "scales"),
    (dict(scales=z(6, 4)[:, ::2]), "scales"), (dict(offsets=z(6, 4)), "offsets must be"), (dict(x=z(3, 64)), "x must be"), (dict(x=odd(W4["x"])), "multiple of 8"),
    (dict(x=z(17, 128), out=z(17, 6)), "at most 16"), (dict(w=z(6, 128, dtype=U8)[:, ::2]), "weight must be"), (dict(out=z(3, 3)), "out must be"),
    (dict(gated=1), "out must be"), (dict(w=z(5, 64, dtype=U8), scales=z(5, 2), out=z(3, 2), gated=1), "even number of rows"),
    (dict(w=z(2, 16448, dtype=U8), scales=z(2, 257), x=z(1, 32896), out=z(1, 2)), "at most 32768")])
def test_gemv_w4(change, match):
    refused("pk_gemv_w4", list({**W4, **change}.values()), match)


def test_operators_refuse_host_tensors():
    from pariskv_b200 import ops
    for f in (lambda: ops.tree_attention(TREE["q"], TREE["k"], TREE["v"], TREE["dk"], TREE["dv"], TREE["mask"].bool(), TREE["lengths"]),
              lambda: ops.block_bounds(BOUNDS["k"]), lambda: ops.select_blocks(SELECT["q"], SELECT["bounds"], SELECT["lengths"], 2),
              lambda: ops.block_attention(ATTEND["q"], ATTEND["k"], ATTEND["v"], ATTEND["blocks"], ATTEND["lengths"]),
              lambda: ops.gemv_w4(W4["w"], W4["scales"], W4["x"])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()


def test_workspace_sizes():
    lib = L.load()
    for rc in (lib.pk_tree_attention_workspace_bytes(8, 61, 32, 8, 131072), lib.pk_block_attention_workspace_bytes(8, 4, 32, 8, 32, 64),
               lib.pk_select_blocks_workspace_bytes(8, 4, 8, 2048)):
        assert 0 < rc < 1 << 32


def test_sizes_that_no_call_takes():
    """Workspace sizes of what would be refused are zero, and a cache ends where 128 rows more still have 31-bit numbers."""
    lib = L.load()
    for T, O, I in ((1, 64, 1 << 41), (1, 64, 32768 + 128), (17, 64, 128), (1, 1 << 40, 128), (0, 64, 128)):
        assert lib.pk_gemv_w4_workspace_bytes(T, O, I, 128, 0) == 0
    long = z(1, 1, 1, 128).expand(2, 2, 2 ** 31 - 100, 128)
    refused("pk_tree_attention", list({**TREE, "k": long, "v": long}.values()), "keys must be")
    refused("pk_block_attention", list({**ATTEND, "k": long, "v": long}.values()), "keys must be")
