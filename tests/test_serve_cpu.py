"""The serving operators' argument checks (no GPU): every refusal comes before
the device is touched, so a call with a stand-in device pointer tests it."""
import ctypes as C

import pytest

import rkcuda as rk

BUF = C.create_string_buffer(1 << 12)
P = (C.addressof(BUF) + 255) // 256 * 256   # 256-byte aligned, never read
DEV = P


def kv8(**over):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, blocks=8, block=16, kv_heads=2, head_size=64)
    f.update(over)
    return rk.KV8(**f)


def refused(rc, *words):
    assert rc == rk.RK_ERR_ARGS
    said = rk.lib().rk_last_error().decode()
    assert all(w in said for w in words), said


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 4),
              dict(k_scale=P + 2), dict(block=0), dict(block=24), dict(block=256), dict(head_size=0), dict(head_size=24),
              dict(head_size=144), dict(head_size=512), dict(kv_heads=0), dict(kv_heads=65536), dict(blocks=0),
              dict(blocks=-1), dict(blocks=1 << 28), dict(blocks=1 << 24, block=128)]


def append(c, **over):
    a = dict(d=DEV, type=rk.ACT_F32, tokens=4, k=P, ks=128, v=P, vs=128, slots=P)
    a.update(over)
    return rk.lib().rk_kv8_append(a["d"], None if c is None else C.addressof(c), a["type"], a["tokens"], a["k"], a["ks"],
                                  a["v"], a["vs"], a["slots"], None)


def attention(c, **over):
    a = dict(d=DEV, type=rk.ACT_BF16, n=2, heads=4, tokens=2, q=P, qs=256, start=None, lens=P, table=P, width=4, scale=0.0,
             window=0, out=P, os=256)
    a.update(over)
    return rk.lib().rk_kv8_attention(a["d"], None if c is None else C.addressof(c), a["type"], a["n"], a["heads"],
                                     a["tokens"], a["q"], a["qs"], a["start"], a["lens"], a["table"], a["width"],
                                     a["scale"], a["window"], a["out"], a["os"], P, 1 << 40, None)


@pytest.mark.parametrize("wrong", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(wrong):
    c = kv8(**wrong)
    refused(append(c), "kv8")
    refused(attention(c), "kv8")
    assert rk.lib().rk_kv8_attention_workspace(DEV, C.addressof(c), 4) == rk.RK_ERR_ARGS


@pytest.mark.parametrize("wrong", [dict(d=None), dict(type=3), dict(type=-1), dict(tokens=-1), dict(k=None), dict(v=None),
                                   dict(slots=None), dict(ks=127), dict(vs=0), dict(ks=-128), dict(k=P + 2),
                                   dict(slots=P + 1), dict(type=rk.ACT_F16, v=P + 1), dict(tokens=(1 << 22) + 1)], ids=str)
def test_append_refuses(wrong):
    refused(append(kv8(), **wrong), "kv8")


def test_append_of_nothing_is_nothing():
    assert append(kv8(), tokens=0, k=None, v=None, slots=None) == rk.RK_OK
    refused(append(None), "null")


@pytest.mark.parametrize("wrong", [dict(d=None), dict(type=7), dict(n=-1), dict(n=rk.MAX_REQUESTS + 1), dict(heads=0),
                                   dict(heads=3), dict(heads=-2), dict(tokens=-1), dict(tokens=1), dict(q=None),
                                   dict(lens=None), dict(table=None), dict(out=None), dict(qs=255), dict(os=1),
                                   dict(width=-1), dict(window=-1), dict(scale=-1.0), dict(scale=float("nan")),
                                   dict(scale=float("inf")), dict(q=P + 1), dict(lens=P + 2), dict(start=P + 2),
                                   dict(table=P + 3), dict(out=P + 1), dict(tokens=(1 << 22) + 1),
                                   dict(tokens=1 << 20, heads=1 << 12, qs=1 << 18, os=1 << 18)], ids=str)
def test_attention_refuses(wrong):
    refused(attention(kv8(), **wrong), "kv8")


def test_attention_of_nothing_is_nothing():
    assert attention(kv8(), n=0) == rk.RK_OK
    assert attention(kv8(), tokens=0, start=P) == rk.RK_OK
    refused(attention(None), "null")


def tables(**over):
    a = dict(d=DEV, n=3, block=16, ctx=P, new=P, free=P, head=None, n_free=5, table=P, width=4, lens=P, start=P, slots=P,
             pos=P, max_tokens=8, info=P)
    a.update(over)
    return rk.lib().rk_page_tables(a["d"], a["n"], a["block"], a["ctx"], a["new"], a["free"], a["head"], a["n_free"],
                                   a["table"], a["width"], a["lens"], a["start"], a["slots"], a["pos"], a["max_tokens"],
                                   a["info"], None)


@pytest.mark.parametrize("wrong", [dict(d=None), dict(n=-1), dict(n=rk.MAX_REQUESTS + 1), dict(block=8), dict(block=48),
                                   dict(ctx=None), dict(new=None), dict(free=None), dict(table=None), dict(lens=None),
                                   dict(start=None), dict(slots=None), dict(pos=None), dict(info=None), dict(n_free=-1),
                                   dict(width=-1), dict(max_tokens=-1), dict(ctx=P + 1), dict(head=P + 2),
                                   dict(slots=P + 2)], ids=str)
def test_tables_refuse(wrong):
    refused(tables(**wrong), "page tables")


def norm(**over):
    a = dict(d=DEV, type=rk.ACT_BF16, rows=2, cols=64, group=32, x=P, xs=64, r=None, rs=64, w=P, eps=1e-5, sum=None, ss=64,
             q=P, scales=P)
    a.update(over)
    return rk.lib().rk_add_rmsnorm_q8(a["d"], a["type"], a["rows"], a["cols"], a["group"], a["x"], a["xs"], a["r"], a["rs"],
                                      a["w"], a["eps"], a["sum"], a["ss"], a["q"], a["scales"], None)


@pytest.mark.parametrize("wrong", [dict(d=None), dict(type=5), dict(rows=-1), dict(cols=0), dict(cols=rk.MAX_COLS + 32),
                                   dict(group=48), dict(group=-1), dict(group=128), dict(x=None), dict(w=None),
                                   dict(q=None), dict(scales=None), dict(xs=63), dict(r=P, rs=8), dict(sum=P, ss=8),
                                   dict(sum=P, ss=128), dict(eps=-1.0), dict(eps=float("nan")), dict(x=P + 1),
                                   dict(w=P + 1), dict(scales=P + 2)], ids=str)
def test_norm_refuses(wrong):
    refused(norm(**wrong), "norm q8")


def test_norm_of_no_rows_is_nothing():
    assert norm(rows=0, x=None, q=None) == rk.RK_OK


def test_w4_refuses():
    L, out = rk.lib(), C.c_void_p()

    def up(d=DEV, rows=4, cols=64, group=32, st=rk.ACT_F32, w=P, s=P, z=None, o=C.addressof(out)):
        return L.rk_w4_upload(d, rows, cols, group, st, w, s, z, o)
    for wrong in (dict(d=None), dict(w=None), dict(s=None), dict(o=None), dict(st=3), dict(rows=0), dict(cols=0),
                  dict(cols=48), dict(cols=rk.MAX_COLS + 32), dict(rows=rk.MAX_ROWS + 1), dict(group=0), dict(group=16),
                  dict(group=48), dict(group=-32), dict(group=128)):
        refused(up(**wrong), "w4")
    zeros = (C.c_uint8 * 8)(*[8] * 7, 16)
    refused(up(z=C.addressof(zeros)), "zero point")
    refused(L.rk_w4_mulvec(None, 1, P, P, 32, rk.ACT_F32, P, 4, None), "w4")
    assert L.rk_w4_bytes(None) == 0
    L.rk_w4_free(None)


def test_device_check_refuses_null():
    refused(rk.lib().rk_device_check(None, None), "null")


def test_tables_refuse_buffers_that_overlap():
    """One call's outputs may not be its inputs (the next step's lengths, the free list's head), nor each other."""
    own = {k: P + 256 * i for i, k in enumerate(("ctx", "new", "free", "head", "table", "lens", "start", "slots", "pos", "info"))}
    ins, outs = ("ctx", "new", "free", "head"), ("table", "lens", "start", "slots", "pos", "info")
    for o in outs:
        for other in ins + outs:
            if other != o:
                refused(tables(**{**own, other: own[o]}), "page tables", "overlap")
    refused(tables(**{**own, "head": own["info"] + 12}), "free_head", "info")
    refused(tables(**{**own, "ctx": own["lens"] - 8}), "ctx_lens", "lens")
    refused(tables(**{**own, "lens": own["ctx"] + 8}), "ctx_lens", "lens")
    refused(tables(**{**own, "free": own["table"] + 4 * 3 * 4 - 4}), "free_pages", "table")


class NoDevice:
    """A device whose tensors are the host's (get_device() is -1): the binding's own checks come first."""
    h = None

    class info:
        index = -1


def test_binding_refuses_shapes():
    """Tensors of a wrong number of dimensions raise RkError like other wrong tensors."""
    import torch
    t = torch.zeros
    kv = rk.PagedKV8(NoDevice, t((2, 2, 16, 32), dtype=torch.int8), t((2, 2, 32, 16), dtype=torch.int8), t((2, 2)), t((2, 2)))
    m = object.__new__(rk.W4Matrix)
    m.index, m.rows, m.cols, m.h = -1, 4, 64, None
    q, i32, x8 = t((1, 4, 32)), dict(dtype=torch.int32), t((1, 64), dtype=torch.int8)
    pages = rk.PageTables.__new__(rk.PageTables)
    pages.dev, pages.index, pages.n = NoDevice, -1, 1
    for call in (lambda: kv.attention(q, t(1, **i32), t(1, **i32)), lambda: kv.attention(q, t((), **i32), t(1, **i32)),
                 lambda: kv.attention(q, t((1, 1, 1), **i32), t(1, **i32)), lambda: kv.attention(q[0], t((1, 1), **i32), t(1, **i32)),
                 lambda: kv.append(q[0], q[0], t(1, **i32)), lambda: kv.append(q[:, :2], q[:, :2], t((1, 1), **i32)),
                 lambda: m.mulvec(x8[0], t((1, 2))), lambda: m.mulvec(x8[0, 0], t((1, 2))), lambda: m.mulvec(x8, t(())),
                 lambda: m.mulvec(x8, t(2)), lambda: m.mulvec(x8, t((1, 0))), lambda: m.mulvec(x8[None], t((1, 2))),
                 lambda: rk.add_rmsnorm_q8(NoDevice, q[0, 0], q[0, 0], 1e-5), lambda: rk.add_rmsnorm_q8(NoDevice, q[0], q[0], 1e-5),
                 lambda: pages.build(t((1, 1), **i32), t(1, **i32), t(1, **i32)),
                 lambda: rk.W4Matrix(NoDevice, t(4, dtype=torch.uint8), t((4, 1))), lambda: rk.W4Matrix(NoDevice, t((4, 16), dtype=torch.uint8), t(4)),
                 lambda: rk.PagedKV8(NoDevice, kv.k[0], kv.v, kv.k_scale, kv.v_scale)):
        with pytest.raises(rk.RkError) as e:
            call()
        assert e.value.code == rk.RK_ERR_ARGS


def test_capture_is_asked_of_the_operators_device():
    """Whether a call is being captured goes by the stream of its own device, not of the current one."""
    from types import SimpleNamespace

    class Fake:
        def __init__(self, now, capturing):
            self.now, self.on = now, capturing
            self._C = SimpleNamespace(_cuda_getDevice=lambda: self.now)
            self.cuda = SimpleNamespace(is_current_stream_capturing=lambda: self.now in self.on, device=self.device)

        def device(self, index):
            fake = self

            class Device:
                def __enter__(self):
                    self.before, fake.now = fake.now, index

                def __exit__(self, *a):
                    fake.now = self.before
            return Device()
    for now in (0, 1):
        for on in ((), (0,), (1,), (0, 1)):
            for index in (0, 1):
                fake = Fake(now, on)
                assert rk._capturing(fake, index) == (index in on)
                assert fake.now == now


@pytest.mark.parametrize("window", [-1, -2 ** 32, 2 ** 31, 2 ** 32, 2 ** 32 + 7])
def test_binding_refuses_windows_past_the_abis_integers(window):
    """A window that 32 bits do not hold is an error, not another window."""
    import torch
    t = torch.zeros
    kv = rk.PagedKV8(NoDevice, t((2, 2, 16, 32), dtype=torch.int8), t((2, 2, 32, 16), dtype=torch.int8), t((2, 2)), t((2, 2)))
    with pytest.raises(rk.RkError) as e:
        kv.attention(t((1, 4, 32)), t((1, 1), dtype=torch.int32), t(1, dtype=torch.int32), window=window)
    assert e.value.code == rk.RK_ERR_ARGS and "window" in str(e.value)
