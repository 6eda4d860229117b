"""Arguments that the operators of a step in 8 bits refuse.  The C ABI checks them before any CUDA call, so that plain host tensors show it."""
import ctypes

import pytest
import torch

from pariskv_b200 import _lib as L
from test_many_arguments import odd, z

I8, I32, I64, F32, E4 = torch.int8, torch.int32, torch.int64, torch.float32, torch.float8_e4m3fn


def call(name, args):
    keep, out = [], []
    for a in args:
        if isinstance(a, dict):
            d = [L.desc(a[k]) for k in ("codes", "scales", "recent")]
            c = L.PkCache8(L.ptr(d[0]), L.ptr(d[1]), L.ptr(d[2]), a["block"])
            keep += [d, c]
            out.append(ctypes.byref(c))
        elif isinstance(a, torch.Tensor):
            d = L.desc(a)
            keep += [a, d]
            out.append(L.ref(d))
        else:
            out.append(a)
    rc = getattr(L.load(), name)(*out)
    return rc, L.load().pk_last_error().decode()


def refused(name, args, match, code=1):
    rc, msg = call(name, args)
    assert rc == code and match in msg, (rc, msg)


CACHE = dict(codes=z(2, 2, 40, 2, 128, dtype=I8), scales=z(2, 2, 3, 2, dtype=F32), recent=z(2, 2, 32, 2, 128), block=16)
APPEND = dict(cache=CACHE, keys=z(2, 3, 2, 128), values=z(2, 3, 2, 128), lengths=z(2, dtype=I32), counts=None, stream=None)
READ = dict(cache=CACHE, lengths=z(2, dtype=I32), rows=None, out=z(2, 2, 40, 2, 128), stream=None)
ATTEND = dict(queries=z(2, 1, 4, 128), cache=CACHE, lengths=z(2, dtype=I32), scale=0.1, out=z(2, 1, 4, 128), lse=None, ws=None, ws_bytes=0, stream=None)
LONG = {**CACHE, "codes": z(1, 1, 1, 2, 128, dtype=I8).expand(2, 2, 20000, 2, 128), "scales": z(1, 1, 1, 2, dtype=F32).expand(2, 2, 1250, 2)}   # a short cache needs no scratch
NORM = dict(a=z(3, 64), residual=z(3, 64), weight=z(64), h=z(3, 64), codes=z(3, 64, dtype=I8), scales=z(3, dtype=F32), eps=1e-6, stream=None)
ROWS = dict(x=z(3, 64), gated=0, codes=z(3, 64, dtype=I8), scales=z(3, dtype=F32), stream=None)
MM = dict(x=z(3, 64, dtype=I8), sx=z(3, dtype=F32), w=z(5, 64, dtype=I8), so=z(5, dtype=F32), out=z(3, 5), stream=None)

CACHES = [
    (dict(codes=z(2, 2, 40, 2, 128, dtype=torch.uint8)), "expected i8 or e4m3"), (dict(codes=z(2, 2, 40, 1, 128, dtype=I8)), "codes must be"), (dict(codes=z(2, 2, 40, 2, 64, dtype=I8)), "codes must be"),
    (dict(codes=z(2, 2, 40, 2, 136, dtype=I8)[..., :128]), "multiples of 16"), (dict(codes=z(2, 2, 40, 2, 256, dtype=I8)[..., ::2]), "unit inner stride"), (dict(block=8), "block must be"),
    (dict(block=48), "block must be"), (dict(scales=z(2, 2, 2, 2, dtype=F32)), "scales must be"), (dict(scales=z(2, 2, 3, 2)), "dtype"), (dict(recent=z(2, 2, 24, 2, 128)), "multiple of block"),
    (dict(recent=z(2, 2, 0, 2, 128)), "recent"), (dict(recent=odd(CACHE["recent"])), "multiples of 8"), (dict(recent=z(2, 1, 32, 2, 128)), "recent must be"), (dict(codes=None), "codes is null"),
    (dict(codes=z(1, 1, 1, 2, 128, dtype=I8).expand(2, 2, 2 ** 31 - 200, 2, 128)), "codes must be")]


@pytest.mark.parametrize("change,match", CACHES)
@pytest.mark.parametrize("name,args", [("pk_cache8_append", APPEND), ("pk_cache8_read", READ), ("pk_cache8_attention", ATTEND)])
def test_caches(name, args, change, match):
    refused(name, list({**args, "cache": {**CACHE, **change}}.values()), match)


@pytest.mark.parametrize("part,to", [("codes", z(1, 2, 40, 2, 128, dtype=I8).expand(2, 2, 40, 2, 128)), ("codes", z(2, 2, 40, 1, 128, dtype=I8).expand(2, 2, 40, 2, 128)),
                                     ("scales", z(2, 2, 1, 2, dtype=F32).expand(2, 2, 3, 2)), ("recent", z(2, 1, 32, 2, 128).expand(2, 2, 32, 2, 128)),
                                     ("codes", z(2 * 2 * 40 * 256, dtype=I8).as_strided((2, 2, 40, 2, 128), (20480, 10240, 128, 128, 1)))])
def test_an_append_into_shared_memory(part, to):
    refused("pk_cache8_append", list({**APPEND, "cache": {**CACHE, part: to}}.values()), "must not share memory")


@pytest.mark.parametrize("change,match", [
    (dict(keys=z(2, 3, 1, 128)), "keys must be"), (dict(keys=z(1, 3, 2, 128)), "keys must be"), (dict(values=z(2, 4, 2, 128)), "shape of keys"), (dict(keys=odd(APPEND["keys"])), "multiples of 8"),
    (dict(keys=z(2, 3, 2, 128, dtype=F32)), "dtype"), (dict(lengths=z(3, dtype=I32)), "lengths must be"), (dict(lengths=z(2, dtype=I64)), "dtype"), (dict(lengths=None), "lengths is null"),
    (dict(counts=z(3, dtype=I32)), "counts must be"), (dict(counts=z(2, dtype=I64)), "dtype")])
def test_append(change, match):
    refused("pk_cache8_append", list({**APPEND, **change}.values()), match)


@pytest.mark.parametrize("change,match", [
    (dict(out=z(2, 2, 41, 2, 128)), "more rows than the cache"), (dict(out=z(2, 1, 40, 2, 128)), "out must be"), (dict(out=z(2, 2, 40, 2, 128, dtype=F32)), "dtype"), (dict(out=odd(READ["out"])), "multiples of 8"),
    (dict(out=z(2, 1, 40, 2, 128).expand(2, 2, 40, 2, 128)), "must not share"), (dict(rows=z(2, 2, 5, dtype=I64)), "rows must be"), (dict(rows=z(2, 2, 40, dtype=I32)), "dtype"),
    (dict(rows=z(2, 40, 2, dtype=I64).transpose(1, 2)), "rows must be")])
def test_read(change, match):
    refused("pk_cache8_read", list({**READ, **change}.values()), match)


@pytest.mark.parametrize("change,match,code", [
    (dict(queries=z(2, 1, 3, 128), out=z(2, 1, 3, 128)), "multiple of the KV heads", 1), (dict(queries=z(2, 1, 4, 64)), "queries must be", 1), (dict(queries=odd(ATTEND["queries"])), "queries must be", 1),
    (dict(queries=z(1, 1, 4, 128), out=z(1, 1, 4, 128)), "codes must be", 1), (dict(out=z(2, 1, 4, 256)[..., ::2]), "out must be", 1), (dict(out=z(2, 1, 2, 128)), "shape of queries", 1),
    (dict(lse=z(2, 1, 2, dtype=F32)), "lse must be", 1), (dict(scale=0.0), "scale must be", 1), (dict(scale=float("nan")), "scale must be", 1), (dict(scale=float("inf")), "scale must be", 1),
    (dict(queries=z(2, 257, 4, 128), out=z(2, 257, 4, 128)), "at most 256", 1), (dict(queries=z(2, 1, 260, 128), out=z(2, 1, 260, 128)), "at most 128", 1), (dict(cache=LONG), "workspace must be", 1), (dict(cache=LONG, ws=4100, ws_bytes=1 << 30), "workspace must be", 1),
    (dict(cache=LONG, ws=4096, ws_bytes=8), "too small", 4), (dict(lengths=z(4, dtype=I32)[::2]), "lengths must be", 1)])
def test_attention(change, match, code):
    refused("pk_cache8_attention", list({**ATTEND, **change}.values()), match, code)


@pytest.mark.parametrize("change,match", [
    (dict(a=z(3, 60), residual=None, weight=z(60), h=z(3, 60), codes=z(3, 60, dtype=I8)), "multiple of 8"), (dict(residual=z(2, 64)), "residual must be"), (dict(weight=z(32)), "weight must be"),
    (dict(h=z(3, 32)), "h_out must be"), (dict(h=z(1, 64).expand(3, 64)), "h_out must be"), (dict(codes=z(3, 64)), "dtype"), (dict(codes=z(1, 64, dtype=I8).expand(3, 64)), "codes must be"),
    (dict(scales=z(4, dtype=F32)), "scales must be"), (dict(a=z(3, 68)[:, :64]), "a must have rows"), (dict(a=z(64, 3).t()), "a must have rows"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(a=z(1, 65544), residual=None, weight=z(65544), h=z(1, 65544), codes=z(1, 65544, dtype=I8), scales=z(1, dtype=F32)), "at most 65536")])
def test_norm(change, match):
    refused("pk_add_rmsnorm_i8", list({**NORM, **change}.values()), match)


@pytest.mark.parametrize("change,match", [
    (dict(gated=1), "codes must be"), (dict(x=z(3, 65), gated=1, codes=z(3, 32, dtype=I8)), "even number"), (dict(x=z(3, 68)[:, :64]), "x must have rows"), (dict(scales=z(3)), "dtype"),
    (dict(x=z(3, 12), codes=z(3, 12, dtype=I8)), "multiple of 8")])
def test_rows(change, match):
    refused("pk_quantize_rows_i8", list({**ROWS, **change}.values()), match)


@pytest.mark.parametrize("change,match", [
    (dict(x=z(3, 72, dtype=I8), w=z(5, 72, dtype=I8)), "multiple of 16"), (dict(w=z(5, 80, dtype=I8)), "as wide as x"), (dict(x=z(3, 72, dtype=I8)[:, :64]), "multiples of 16"),
    (dict(w=z(64, 5, dtype=I8).t()), "unit inner stride"), (dict(x=z(1, 64, dtype=I8).expand(3, 64)), "multiples of 16"), (dict(sx=z(2, dtype=F32)), "x_scales must be"), (dict(so=z(4, dtype=F32)), "weight_scales must be"),
    (dict(so=z(10, dtype=F32)[::2]), "weight_scales must be"), (dict(out=z(3, 6)), "out must be"), (dict(out=z(5, 3).t()), "out must be"), (dict(out=z(1, 5).expand(3, 5)), "out must be"),
    (dict(x=z(3, 64, dtype=torch.uint8)), "dtype"), (dict(x=z(1, 65552, dtype=I8), w=z(1, 65552, dtype=I8)), "at most 65536")])
def test_matmul(change, match):
    refused("pk_matmul_i8", list({**MM, **change}.values()), match)


def test_operators_refuse_host_tensors():
    from pariskv_b200 import ops
    cache = ops.Cache8(**CACHE)
    for f in (lambda: ops.cache8_append(cache, APPEND["keys"], APPEND["values"], APPEND["lengths"]), lambda: ops.cache8_read(cache, READ["lengths"]),
              lambda: ops.cache8_attention(ATTEND["queries"], cache, ATTEND["lengths"]), lambda: ops.add_rmsnorm_i8(NORM["a"], None, NORM["weight"]), lambda: ops.quantize_rows_i8(ROWS["x"]),
              lambda: ops.matmul_i8(MM["x"], MM["sx"], MM["w"], MM["so"])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()


def test_workspace_sizes():
    lib = L.load()
    assert 0 < lib.pk_cache8_attention_workspace_bytes(8, 4, 32, 8, 131072) < 1 << 30
    assert lib.pk_cache8_attention_workspace_bytes(8, 300, 32, 8, 131072) == 0
    assert lib.pk_cache8_attention_workspace_bytes(1, 1, 32, 8, 256) == 0
