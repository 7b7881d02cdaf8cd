"""The C ABI and argument checks of the linear-attention and state-page calls,
without a GPU."""
from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from conftest import ROOT, graft, has_gpu

HEADER = ROOT / "include" / "gdn_b200.h"
BASE = 0x7F0000000000


def test_struct_layout_matches_header(pkg, tmp_path):
    L = pkg._lib
    pairs = [("lin_decode_args_t", L.LinDecodeArgs), ("lin_prefill_args_t", L.LinPrefillArgs),
             ("pages_pool_t", L.PagesPool), ("pages_args_t", L.PagesArgs)]
    body = ["#include <stdio.h>", f'#include "{HEADER}"', "int main(void){"]
    expect = []
    for c, py in pairs:
        body.append(f'printf("%zu\\n", sizeof({c}));')
        expect.append(ctypes.sizeof(py))
        for f, _ in py._fields_:
            body.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            expect.append(getattr(py, f).offset)
    body += ['printf("%d\\n%d\\n", PAGES_MAX_POOLS, PAGES_MAX_PAGES);', "return 0;}"]
    expect += [L.PAGES_MAX_POOLS, L.PAGES_MAX_PAGES]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(body))
    subprocess.run(["gcc", "-std=c99", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == expect


def test_packed_arguments_match_the_structs(pkg):
    """The bytes that a call passes are those of the ctypes struct, field by field."""
    lin, pages = _lin(), graft.submodule("pages")
    for packed, cls in [(lin._DECODE, pkg._lib.LinDecodeArgs), (lin._PREFILL, pkg._lib.LinPrefillArgs),
                        (pages._CALLS["fork"], pkg._lib.PagesArgs)]:
        values = [i + 1 for i in range(len(cls._fields_))]
        a = cls.from_buffer_copy(packed.pack(*values))
        got = [getattr(a, f) for f, _ in cls._fields_]
        got = [ctypes.cast(x, ctypes.c_void_p).value if isinstance(x, ctypes.POINTER(pkg._lib.PagesPool)) else x
               for x in got]
        assert got == values


def test_values_beyond_a_field_are_refused(pkg):
    for scale in (1e39, float("inf"), float("nan")):
        with pytest.raises(pkg.GDNError, match="scale"):
            _lin()._decode_args(**{**_dec(), "scale": scale})
        with pytest.raises(pkg.GDNError, match="scale"):
            _lin()._prefill_args(**{**_pre(), "scale": scale})
    with pytest.raises(pkg.GDNError, match="pages_copy_launch"):
        graft.submodule("pages")._CALLS["copy"].pack(0, 0, 1, 0, 0, 1 << 31, *[0] * 7)


def decode_args(pkg, **over):
    a = pkg._lib.LinDecodeArgs()
    for i, name in enumerate(("q", "k", "v", "g", "state_in", "o")):
        setattr(a, name, BASE + i * (1 << 32))
    a.state_out = a.state_in
    B, Hqk, Hv, d = 4, 2, 4, 128
    a.q_sb, a.q_sh, a.k_sb, a.k_sh = Hqk * d, d, Hqk * d, d
    a.v_sb, a.v_sh, a.o_sb, a.o_sh = Hv * d, d, Hv * d, d
    a.g_sb, a.g_sh = Hv, 1
    a.state_in_sp = a.state_out_sp = Hv * d * d
    a.B, a.Hqk, a.Hv, a.dk, a.dv, a.pages = B, Hqk, Hv, d, d, B
    a.io_dtype, a.scale = 1, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    ({"q": 0}, 1), ({"o": 0}, 1), ({"state_in": 0}, 1),
    ({"Hv": 3}, 2), ({"dk": 96}, 2), ({"dv": 96}, 2), ({"dv": 0}, 2), ({"B": 0}, 2),
    ({"pages": 3}, 2),                        # fewer pages than rows, no index
    ({"pages": 0, "index": BASE}, 2),
    ({"state_in_sp": 4 * 128 * 128 - 4}, 2),  # pages overlap
    ({"state_out_sp": 5 * 128 * 128}, 2),     # in place with two strides
    ({"state_out": BASE + 4 * (1 << 32) + 4096}, 2),
    ({"io_dtype": 0}, 4), ({"g_dtype": 7}, 4), ({"gate_kind": 5}, 4),
    ({"q": BASE + 8}, 3), ({"v_sh": 100}, 3), ({"state_in_sp": 4 * 128 * 128 + 2}, 3),
    ({"o_sb": 0}, 2), ({"o_sh": 0}, 2),
])
def test_decode_refuses(pkg, over, code):
    a = decode_args(pkg, **over)
    assert pkg._lib.load().lin_decode_launch(ctypes.byref(a), None) == code


def prefill_args(pkg, **over):
    a = pkg._lib.LinPrefillArgs()
    for i, name in enumerate(("q", "k", "v", "g", "final_state", "o")):
        setattr(a, name, BASE + i * (1 << 32))
    B, T, Hqk, Hv, d = 2, 70, 2, 4, 128
    a.q_sb, a.q_st, a.q_sh = T * Hqk * d, Hqk * d, d
    a.k_sb, a.k_st, a.k_sh = T * Hqk * d, Hqk * d, d
    a.v_sb, a.v_st, a.v_sh = T * Hv * d, Hv * d, d
    a.o_sb, a.o_st, a.o_sh = T * Hv * d, Hv * d, d
    a.g_sb, a.g_st, a.g_sh = T * Hv, Hv, 1
    a.final_sp = a.initial_sp = Hv * d * d
    a.B, a.T, a.Hqk, a.Hv, a.dk, a.dv, a.pages = B, T, Hqk, Hv, d, d, B
    a.io_dtype, a.scale = 1, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    ({"k": 0}, 1), ({"final_state": 0}, 1),
    ({"Hqk": 3}, 2), ({"dk": 256}, 2), ({"dv": 32}, 2), ({"T": 0}, 2), ({"B": 0}, 2), ({"B": 70000}, 2),
    ({"pages": 1}, 2), ({"final_sp": 64}, 2), ({"q_st": -256}, 2), ({"o_st": 0}, 2), ({"k_sh": 0}, 2),
    ({"initial_state": BASE + 4 * (1 << 32) + 64}, 2),
    ({"initial_state": BASE + 4 * (1 << 32), "initial_sp": 5 * 128 * 128}, 2),
    ({"io_dtype": 0}, 4), ({"g_dtype": -1}, 4),
    ({"o": BASE + 4}, 3), ({"k_st": 260}, 3), ({"final_sp": 4 * 128 * 128 + 1}, 3),
])
def test_prefill_refuses(pkg, over, code):
    a = prefill_args(pkg, **over)
    assert pkg._lib.load().lin_prefill_launch(ctypes.byref(a), None) == code


def pages_args(pkg, pool=None, **over):
    L = pkg._lib
    pools = (L.PagesPool * 1)(pool or (BASE, 4096, 4096))
    M = 1 << 24
    a = L.PagesArgs(pools, 1, 8, BASE, BASE, 4, BASE + M, BASE + 2 * M, BASE + 3 * M, BASE + 4 * M,
                    BASE + 5 * M, 4096, None)
    for k, v in over.items():
        setattr(a, k, v)
    a._keep = pools
    return a


@pytest.mark.parametrize("fn", ["copy", "fork", "compact"])
@pytest.mark.parametrize("over,code", [
    ({"pages": 0}, 2), ({"pages": (1 << 19) + 1}, 2), ({"n": -1}, 2), ({"n_pools": 65}, 2),
    ({"pool": (0, 4096, 4096)}, 1), ({"pool": (BASE, 4080, 4096)}, 2), ({"pool": (BASE, 4096, 4088)}, 3),
    ({"pool": (BASE, 4100, 4096)}, 3), ({"pool": (BASE + 8, 4096, 4096)}, 3),
    ({"dst": 0}, 1),
    # (small calls need no workspace)
    ({"pages": 5000, "n": 3000, "workspace": 0}, 7), ({"pages": 5000, "n": 3000, "workspace_bytes": 12}, 7),
    ({"pages": 5000, "n": 3000, "workspace": BASE + 2, "workspace_bytes": 1 << 20}, 3),
])
def test_pages_refuse(pkg, fn, over, code):
    a = pages_args(pkg, **over)
    assert getattr(pkg._lib.load(), f"pages_{fn}_launch")(ctypes.byref(a), None) == code


@pytest.mark.parametrize("fn,over", [
    ("fork", {"dst": BASE + (1 << 24) + 4}),       # entries and results share memory
    ("fork", {"used_out": BASE + 16}),             # flags shifted against themselves
    ("fork", {"dst": BASE + 16}), ("fork", {"src": BASE}),
    ("free", {"src": BASE + 8}),
    ("compact", {"dst": BASE + (1 << 24) + 4}), ("compact", {"remap": BASE}), ("compact", {"count": BASE + 3 * (1 << 24)}),
    ("compact", {"src": BASE + 8}),
])
def test_pages_refuse_shared_memory(pkg, fn, over):
    a = pages_args(pkg, **over)
    assert getattr(pkg._lib.load(), f"pages_{fn}_launch")(ctypes.byref(a), None) == 2


def test_pages_workspace(pkg):
    L = pkg._lib.load()
    assert L.pages_workspace_size(ctypes.byref(pages_args(pkg, pages=2048, n=2048))) == 0
    assert L.pages_workspace_size(ctypes.byref(pages_args(pkg, pages=2049, n=4))) == 4 * 2049
    assert L.pages_workspace_size(ctypes.byref(pages_args(pkg, pages=8, n=3000, remap=0))) == 4 * 3000


def test_pages_refuse_missing_flags(pkg):
    L = pkg._lib.load()
    for fn in ("fork", "free", "compact"):
        a = pages_args(pkg, used=0)
        assert getattr(L, f"pages_{fn}_launch")(ctypes.byref(a), None) == 1
    a = pages_args(pkg, remap=0)
    assert L.pages_compact_launch(ctypes.byref(a), None) == 1


@pytest.mark.skipif(has_gpu(), reason="checks the no-device path")
def test_sound_calls_without_gpu_report_no_device(pkg):
    L = pkg._lib.load()
    assert L.lin_decode_launch(ctypes.byref(decode_args(pkg)), None) == 6
    assert L.lin_prefill_launch(ctypes.byref(prefill_args(pkg)), None) in (6, 7)
    for fn in ("copy", "fork", "free", "compact"):
        assert getattr(L, f"pages_{fn}_launch")(ctypes.byref(pages_args(pkg)), None) == 6


def test_null_arguments(pkg):
    L = pkg._lib.load()
    for fn in ("lin_decode_launch", "lin_prefill_launch", "pages_copy_launch", "pages_fork_launch",
               "pages_free_launch", "pages_compact_launch"):
        assert getattr(L, fn)(None, None) == 1
    assert L.pages_workspace_size(None) == 0 and L.lin_prefill_workspace_size(None) == 0


# ------------------------------------------------------- the Python layer's checks


def _lin():
    return graft.submodule("lin")


def _dec(B=2, Hqk=1, Hv=2, d=64):
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    return {"q": z(B, Hqk, d), "k": z(B, Hqk, d), "v": z(B, Hv, d), "g": z(B, Hv, t=torch.float32),
            "state": z(B, Hv, d, d, t=torch.float32), "state_out": z(B, Hv, d, d, t=torch.float32),
            "out": z(B, Hv, d), "index": None, "scale": 1.0, "gate": "log"}


@pytest.mark.parametrize("over", [
    {"k": torch.zeros(2, 2, 64, dtype=torch.bfloat16)}, {"k": torch.zeros(2, 1, 64)},
    {"v": torch.zeros(3, 2, 64, dtype=torch.bfloat16)}, {"g": torch.zeros(2, 3)}, {"g": torch.zeros(2, 2, 64)},
    {"g": torch.zeros(2, 2, dtype=torch.float64)},
    {"out": torch.zeros(2, 2, 32, dtype=torch.bfloat16)}, {"out": torch.zeros(2, 64, 2, dtype=torch.bfloat16).mT},
    {"state": torch.zeros(2, 2, 64, 64, dtype=torch.float16)}, {"state": torch.zeros(2, 2, 64, 64).mT},
    {"state": torch.zeros(3, 2, 64, 64)}, {"state_out": torch.zeros(1, 2, 64, 64)},
    {"index": torch.zeros(2, dtype=torch.int64)}, {"index": torch.zeros(3, dtype=torch.int32)}, {"gate": "exp"},
])
def test_decode_arguments(pkg, over):
    lin = _lin()
    lin._decode_args(**_dec())
    with pytest.raises(pkg.GDNError):
        lin._decode_args(**{**_dec(), **over})


def _pre(B=2, T=5, Hqk=1, Hv=2, d=64):
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    return {"q": z(B, T, Hqk, d), "k": z(B, T, Hqk, d), "v": z(B, T, Hv, d), "g": z(B, T, Hv, t=torch.float32),
            "initial_state": None, "final_state": z(B, Hv, d, d, t=torch.float32), "out": z(B, T, Hv, d),
            "cu_seqlens": None, "index": None, "scale": 1.0}


@pytest.mark.parametrize("over", [
    {"k": torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16)}, {"v": torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)},
    {"g": torch.zeros(2, 5, 1)}, {"g": torch.zeros(3)}, {"out": torch.zeros(2, 5, 2, 64)},
    {"final_state": torch.zeros(3, 2, 64, 64)}, {"initial_state": torch.zeros(1, 2, 64, 64)},
    {"cu_seqlens": torch.zeros(3, dtype=torch.int32)},  # packed needs a batch of one
    {"cu_seqlens": torch.zeros(3, dtype=torch.int64)}, {"index": torch.zeros(1, dtype=torch.int32)},
])
def test_prefill_arguments(pkg, over):
    lin = _lin()
    lin._prefill_args(**_pre())
    with pytest.raises(pkg.GDNError):
        lin._prefill_args(**{**_pre(), **over})


def test_pools(pkg):
    pages = graft.submodule("pages")
    pages._pools([torch.zeros(4, 8), torch.zeros(4, 2, 8)[:, 1]])
    for bad in ([torch.zeros(4, 8), torch.zeros(5, 8)], [torch.zeros(4, 8, 2).mT], [torch.zeros(4)],
                [torch.zeros(2, 8)] * 65):
        with pytest.raises(pkg.GDNError):
            pages._pools(bad)


def test_cpu_tensors_are_refused(pkg):
    d, p, flags = _dec(), _pre(), torch.zeros(4, dtype=torch.int32)
    pool = torch.zeros(4, 64)
    for call in (lambda: pkg.lin_decode(*(d[x] for x in ("q", "k", "v", "g", "state"))),
                 lambda: pkg.lin_prefill(*(p[x] for x in ("q", "k", "v", "g"))),
                 lambda: pkg.pages_copy(pool, flags, flags), lambda: pkg.pages_fork(pool, flags, flags),
                 lambda: pkg.pages_alloc(flags, 1), lambda: pkg.pages_free(flags, flags),
                 lambda: pkg.pages_compact(pool, flags)):
        with pytest.raises(pkg.GDNError):
            call()


# ------------------------------------------------------- strides of axes of one entry


ONE_D = {"B": 1, "Hqk": 1, "Hv": 1, "pages": 1, "state_in_sp": 1, "state_out_sp": 3,
         **{x: 1 for x in ("q_sb", "q_sh", "k_sb", "k_sh", "v_sb", "v_sh", "o_sb", "o_sh")}}
ONE_P = {"B": 1, "T": 1, "Hqk": 1, "Hv": 1, "pages": 1, "final_sp": 1, "initial_sp": 3,
         **{x + y: 1 for x in ("q_s", "k_s", "v_s", "o_s") for y in "bth"}}


@pytest.mark.skipif(has_gpu(), reason="checks the no-device path")
def test_strides_of_axes_of_one_entry_are_free(pkg):
    L = pkg._lib.load()
    assert L.lin_decode_launch(ctypes.byref(decode_args(pkg, **ONE_D)), None) == 6
    assert L.lin_prefill_launch(ctypes.byref(prefill_args(pkg, **ONE_P)), None) == 6
    # packed: one batch, whatever the number of sequences
    a = prefill_args(pkg, cu_seqlens=BASE, q_sb=1, k_sb=-3, v_sb=5, o_sb=0)
    assert L.lin_prefill_launch(ctypes.byref(a), None) == 6


@pytest.mark.parametrize("one,over", [(ONE_D, {"B": 2, "pages": 2, "state_in_sp": 1 << 16, "state_out_sp": 1 << 16}), (ONE_D, {"Hv": 2})])
def test_decode_strides_of_longer_axes_are_checked(pkg, one, over):
    a = decode_args(pkg, **{**one, **over})
    assert pkg._lib.load().lin_decode_launch(ctypes.byref(a), None) == 3


@pytest.mark.parametrize("over", [{"B": 2, "pages": 2, "final_sp": 1 << 16}, {"T": 2}, {"Hv": 2}])
def test_prefill_strides_of_longer_axes_are_checked(pkg, over):
    a = prefill_args(pkg, **{**ONE_P, **over})
    assert pkg._lib.load().lin_prefill_launch(ctypes.byref(a), None) == 3


# ------------------------------------------------------- pools between one another

PAGE = 4 * 128 * 128  # elements of a page of decode_args and prefill_args
IN = BASE + 4 * (1 << 32)


@pytest.mark.parametrize("sp,shift,ok", [
    (2 * PAGE, PAGE, True), (3 * PAGE, 2 * PAGE, True), (3 * PAGE, PAGE, True), (2 * PAGE, -PAGE, True),
    (3 * PAGE, 7 * PAGE, True),                             # another layer, some pages on
    (PAGE, 4 * PAGE, True), (PAGE, -4 * PAGE, True),        # end to end
    (PAGE, PAGE, False), (3 * PAGE, 3 * PAGE, False),       # the next page of the same layer
    (2 * PAGE, PAGE - 4, False), (2 * PAGE, PAGE + 4, False), (2 * PAGE + 8, PAGE + 4, True),
    (2 * PAGE, 4, False),
])
def test_pools_that_share_memory(pkg, sp, shift, ok):
    L = pkg._lib.load()
    if ok and has_gpu():
        pytest.skip("checks the no-device path")
    a = decode_args(pkg, state_in_sp=sp, state_out_sp=sp, state_out=IN + 4 * shift)
    assert L.lin_decode_launch(ctypes.byref(a), None) == (6 if ok else 2)
    a = prefill_args(pkg, B=4, T=7, pages=4, initial_sp=sp, final_sp=sp, initial_state=IN + 4 * shift, final_state=IN)
    assert L.lin_prefill_launch(ctypes.byref(a), None) == (6 if ok else 2)


def test_pools_of_unlike_strides_must_lie_apart(pkg):
    L = pkg._lib.load()
    a = decode_args(pkg, state_in_sp=2 * PAGE, state_out_sp=4 * PAGE, state_out=IN + 4 * PAGE)
    assert L.lin_decode_launch(ctypes.byref(a), None) == 2
    a = prefill_args(pkg, initial_sp=4 * PAGE, final_sp=2 * PAGE, initial_state=IN + 4 * PAGE, final_state=IN)
    assert L.lin_prefill_launch(ctypes.byref(a), None) == 2


def test_workspace_is_asked_for_on_the_tensors_device(pkg, monkeypatch):
    lin, at, asked = _lin(), [0], []

    class On:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, at[0] = at[0], self.dev

        def __exit__(self, *_):
            at[0] = self.before

    class Library:
        @staticmethod
        def lin_prefill_workspace_size(_):
            asked.append(at[0])
            return 7

    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(lin._lib, "load", lambda: Library)
    args = lin._prefill_args(**_pre())
    assert lin._prefill_workspace(args, 3) == lin._prefill_workspace(args, 0) == lin._prefill_workspace(args) == 7
    assert asked == [3, 0, 0] and at == [0]


def test_small_page_calls_need_no_workspace(pkg):
    """What lets a call of few pages and entries go without asking for the size."""
    small = graft.submodule("pages")._SMALL
    L = pkg._lib.load()
    for n in (1, small):
        for pages in (1, small):
            for remap in (0, BASE):
                a = pages_args(pkg, pages=pages, n=n, remap=remap)
                assert L.pages_workspace_size(ctypes.byref(a)) == 0
    assert L.pages_workspace_size(ctypes.byref(pages_args(pkg, pages=1, n=small + 1, remap=0))) > 0
    assert L.pages_workspace_size(ctypes.byref(pages_args(pkg, pages=small + 1, n=1))) > 0
