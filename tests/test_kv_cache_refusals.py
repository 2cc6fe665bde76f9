"""What the entry points of the paged cache refuse, before they touch a device (no GPU needed: a call that passes its checks here fails
for want of one, with another status)."""
import ctypes as C

import pytest

from rai_amd import _lib
from rai_amd.hip import HipTensor

ARG, SHAPE, STRIDE, DTYPE, UNSUPPORTED = -6, -2, -3, -1, -7


class Place:
    """Memory nobody reads: an address."""
    at = 1 << 40

    def __init__(self, ptr=None):
        if ptr is None:
            Place.at += 1 << 36
            ptr = Place.at
        self.ptr, self.dev = ptr, 0


def t(dtype, *shape, strides=None, offset=0, ptr=None):
    return HipTensor(Place(ptr), dtype, shape, strides, offset)


def status(name, *args):
    args = [a.desc() if isinstance(a, HipTensor) else a for a in args]
    return getattr(_lib.load(), name)(0, *(C.byref(a) if isinstance(a, _lib.TensorDesc) else a for a in args))


def cache(pages=9, heads=2, page=16, f=64):
    return dict(format=0, k=t("u8", pages, heads, page, f), v=t("u8", pages, heads, f, page), k_scale=t("f32", pages, heads), v_scale=t("f32", pages, heads))


def plan(**over):
    a = dict(lens=t("i64", 3), add=t("i64", 3), free=t("u32", 20), taken=t("i64", 1), tables=t("u32", 3, 8), page=16, out_tables=t("u32", 3, 8), out_lens=t("i64", 3),
             out_taken=t("i64", 1), starts=t("i64", 4), positions=t("i64", 40), runs=t("u32", 4, 8))
    a.update(over)
    return status("rai_hip_kv_plan", *a.values())


def rope(**over):
    a = dict(x=t("bf16", 5, 4, 64), positions=t("i64", 5), frequencies=t("f64", 32), interleaved=0, inverse=0, magnitude=1.0, out=t("bf16", 5, 4, 64))
    a.update(over)
    return status("rai_hip_rope_positions", *a.values())


def append(**over):
    a = dict(new_k=t("bf16", 5, 2, 60), new_v=t("bf16", 5, 2, 60), runs=t("u32", 4, 5), **cache())
    a.update(over)
    return status("rai_hip_kv_append", *a.values())


def attention(**over):
    a = dict(q=t("bf16", 5, 4, 60), tables=t("u32", 3, 8), starts=t("i64", 4), lens=t("i64", 3), **cache(), scale=1.0, window=0, out=t("bf16", 5, 4, 60))
    a.update(over)
    return status("rai_hip_kv_attention", *a.values())


def needs_no_gpu():
    n = C.c_int(0)
    return _lib.load().rai_hip_device_count(C.byref(n)) != 0 or n.value == 0


@pytest.mark.skipif(not needs_no_gpu(), reason="addresses here are nobody's: with a GPU a call that passes would use them")
def test_the_unchanged_calls_pass_their_checks():
    assert [f() for f in (plan, rope, append, attention)] == [-5] * 4   # no device


@pytest.mark.parametrize("want,over", [
    (DTYPE, dict(lens=t("u32", 3))), (DTYPE, dict(tables=t("i64", 3, 8))), (DTYPE, dict(runs=t("i64", 4, 8))), (DTYPE, dict(free=t("i64", 20))),
    (ARG, dict(page=24)), (ARG, dict(page=8)), (ARG, dict(page=512)), (ARG, dict(page=0)), (ARG, dict(page=-16)),
    (SHAPE, dict(add=t("i64", 2))), (SHAPE, dict(starts=t("i64", 3))), (SHAPE, dict(out_tables=t("u32", 3, 9))), (SHAPE, dict(taken=t("i64", 2))),
    (SHAPE, dict(runs=t("u32", 4, 7))), (SHAPE, dict(runs=t("u32", 3, 8))), (DTYPE, dict(positions=t("i64", 40, strides=(2,)))),
    (STRIDE, dict(tables=t("u32", 3, 8, strides=(1, 3)))), (STRIDE, dict(out_tables=t("u32", 3, 8, strides=(4, 1)))),
    (STRIDE, dict(runs=t("u32", 4, 8, strides=(16, 1)))),
    (UNSUPPORTED, dict(lens=t("i64", 4097), add=t("i64", 4097), tables=t("u32", 4097, 8), out_tables=t("u32", 4097, 8), out_lens=t("i64", 4097), starts=t("i64", 4098), runs=t("u32", 4, 40))),
])
def test_plan_refuses(want, over):
    assert plan(**over) == want


def test_plan_refuses_outputs_over_inputs():
    lens, tables = t("i64", 3), t("u32", 3, 8)
    assert plan(lens=lens, out_lens=lens) == ARG
    assert plan(tables=tables, out_tables=HipTensor(tables.buf, "u32", (3, 8), offset=8)) == ARG
    assert plan(tables=tables, out_tables=HipTensor(tables.buf, "u32", (3, 8), (9, 1))) == ARG
    assert plan(out_lens=lens, positions=HipTensor(lens.buf, "i64", (40,), offset=2)) == ARG
    assert plan(free=tables, tables=tables) == SHAPE


@pytest.mark.parametrize("want,over", [
    (DTYPE, dict(x=t("f64", 5, 4, 64))), (DTYPE, dict(out=t("f32", 5, 4, 64))), (DTYPE, dict(positions=t("u32", 5))), (DTYPE, dict(frequencies=t("f32", 32))),
    (SHAPE, dict(x=t("bf16", 5, 256))), (SHAPE, dict(out=t("bf16", 5, 4, 32))), (SHAPE, dict(positions=t("i64", 4))), (SHAPE, dict(frequencies=t("f64", 33))),
    (STRIDE, dict(x=t("bf16", 5, 4, 64, strides=(512, 128, 2)))), (SHAPE, dict(out=t("bf16", 5, 4, 64, strides=(512, 64, 1)))),
    (UNSUPPORTED, dict(x=t("bf16", 5, 4, 1040), out=t("bf16", 5, 4, 1040)))])
def test_rope_refuses(want, over):
    assert rope(**over) == want


def test_rope_refuses_to_work_in_place():
    x = t("bf16", 5, 4, 64)
    assert rope(x=x, out=x) == ARG


@pytest.mark.parametrize("want,args", [(ARG, (0.0, 0, 1, 4, 8192)), (ARG, (1e4, -1.0, 1, 4, 8192)), (ARG, (1e4, 8.0, 4, 4, 8192)), (ARG, (1e4, 8.0, 0, 4, 8192)),
                                       (ARG, (1e4, 8.0, 1, 4, 0)), (ARG, (float("nan"), 0, 1, 4, 8192)), (ARG, (1e4, float("nan"), 1, 4, 8192))])
def test_frequencies_refuse(want, args):
    assert status("rai_hip_rope_frequencies", *map(float, args), t("f64", 32)) == want


def test_frequencies_are_f64():
    assert status("rai_hip_rope_frequencies", 1e4, 0.0, 1.0, 4.0, 8192.0, t("f32", 32)) == DTYPE


BAD_CACHE = [
    (ARG, dict(format=2)), (ARG, dict(format=-1)), (DTYPE, dict(k=t("i64", 9, 2, 16, 64))), (DTYPE, dict(k_scale=t("bf16", 9, 2))),
    (SHAPE, dict(v=t("u8", 9, 2, 16, 64))), (SHAPE, dict(v=t("u8", 8, 2, 64, 16))), (SHAPE, dict(k_scale=t("f32", 9, 1), v_scale=t("f32", 9, 1))), (SHAPE, dict(v_scale=t("f32", 2, 9))),
    (SHAPE, dict(k=t("u8", 9, 2, 24, 64), v=t("u8", 9, 2, 64, 24))), (SHAPE, dict(k=t("u8", 9, 2, 16, 60), v=t("u8", 9, 2, 60, 16))),
    (SHAPE, dict(k=t("u8", 9, 2, 16, 272), v=t("u8", 9, 2, 272, 16))), (SHAPE, dict(k=t("u8", 9, 2, 16, 80), v=t("u8", 9, 2, 80, 16))),
    (STRIDE, dict(k=t("u8", 9, 2, 16, 64, strides=(4096, 1024, 64, 1)))), (STRIDE, dict(v=t("u8", 9, 2, 64, 16, offset=8))),
    (SHAPE, dict(k=t("u8", 0, 2, 16, 64), v=t("u8", 0, 2, 64, 16), k_scale=t("f32", 0, 2), v_scale=t("f32", 0, 2)))]


@pytest.mark.parametrize("want,over", BAD_CACHE + [
    (DTYPE, dict(new_k=t("f64", 5, 2, 60), new_v=t("f64", 5, 2, 60))), (DTYPE, dict(new_v=t("f16", 5, 2, 60))), (DTYPE, dict(runs=t("i64", 4, 5))),
    (SHAPE, dict(new_v=t("bf16", 4, 2, 60))), (SHAPE, dict(new_k=t("bf16", 5, 4, 60), new_v=t("bf16", 5, 4, 60))), (SHAPE, dict(runs=t("u32", 5, 4))),
    (SHAPE, dict(new_k=t("bf16", 5, 2, 48), new_v=t("bf16", 5, 2, 48))), (STRIDE, dict(new_k=t("bf16", 5, 2, 60, strides=(240, 120, 2))))])
def test_append_refuses(want, over):
    assert append(**over) == want


def test_append_refuses_a_cache_over_itself_or_its_inputs():
    c, new = cache(), t("bf16", 5, 2, 60)
    assert append(v_scale=c["k_scale"], k_scale=c["k_scale"]) == ARG
    assert append(new_k=new, k=HipTensor(new.buf, "u8", (9, 2, 16, 64))) == ARG


@pytest.mark.parametrize("want,over", BAD_CACHE + [
    (DTYPE, dict(q=t("f64", 5, 4, 60), out=t("f64", 5, 4, 60))), (DTYPE, dict(out=t("f32", 5, 4, 60))), (DTYPE, dict(tables=t("i64", 3, 8))), (DTYPE, dict(lens=t("u32", 3))),
    (SHAPE, dict(q=t("bf16", 5, 3, 60), out=t("bf16", 5, 3, 60))), (SHAPE, dict(out=t("bf16", 5, 4, 64))), (SHAPE, dict(starts=t("i64", 3))), (SHAPE, dict(lens=t("i64", 4))),
    (SHAPE, dict(out=t("bf16", 5, 4, 60, strides=(256, 64, 1)))), (STRIDE, dict(q=t("bf16", 5, 4, 60, strides=(480, 120, 2)))), (STRIDE, dict(tables=t("u32", 3, 8, strides=(1, 3)))),
    (ARG, dict(window=-1)), (UNSUPPORTED, dict(tables=t("u32", 3, 1 << 27))), (UNSUPPORTED, dict(q=t("bf16", 1 << 26, 4, 60), out=t("bf16", 1 << 26, 4, 60)))])
def test_attention_refuses(want, over):
    assert attention(**over) == want


def test_attention_refuses_an_output_over_an_input():
    q = t("bf16", 5, 4, 60)
    assert attention(q=q, out=q) == ARG


def test_attention_refuses_more_tiles_than_a_launch_holds():
    """2^22 tiles of a head, of two heads."""
    assert attention(q=t("bf16", 1 << 25, 4, 60), out=t("bf16", 1 << 25, 4, 60)) == UNSUPPORTED
