"""Forked, cut and compacted sequences, rotary tables, refusals of the C entries: what needs no GPU."""
import ctypes
import math

import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.paged import PageTable, copy_pages, draft_tree
from VAR_Q.rotary import Rotary


def table(pages=8, size=16, **lens):
    t = PageTable(pages, size)
    for s, n in lens.items():
        t.add(s)
        t.extend([s], [n], "cpu")
    return t


def test_fork_shares_full_pages():
    t = table(a=40, b=32)
    pages = t._pages["a"][:]
    src, dst = t.fork(["a", "a", "b"], ["x", "y", "z"], "cpu")
    assert src.tolist() == [pages[2]] * 2 and len(set(dst.tolist())) == 2 and t.free_pages == 1
    assert t._pages["x"] == pages[:2] + [dst[0].item()] and t._pages["z"] == t._pages["b"] and t.length("y") == 40
    t.remove("a")
    assert t.free_pages == 2                                             # the shared ones stay
    t.extend(["x", "z"], [5, 1], "cpu")
    assert t._pages["z"][:2] == t._pages["b"] and len(t._pages["z"]) == 3
    for s in ("x", "y", "z", "b"):
        t.remove(s)
    assert t.free_pages == 8 and not any(t._owners)


def test_fork_refuses_and_takes_nothing():
    t = table(pages=4, a=40)
    with pytest.raises(RuntimeError, match="2 pages needed, 1 are free"):
        t.fork(["a", "a"], ["x", "y"], "cpu")
    for args in ((["a"], ["a"]), (["a"], ["x", "y"]), (["a", "a"], ["x", "x"])):
        with pytest.raises(ValueError):
            t.fork(*args, "cpu")
    with pytest.raises(KeyError):
        t.fork(["nobody"], ["x"], "cpu")
    assert t.free_pages == 1 and "x" not in t and t._owners == [1, 1, 1, 0]
    assert t.fork([], [], "cpu")[0].shape == (0,)


def test_accept_moves_and_gives_back():
    t = table(a=14, b=3)
    t.extend(["a", "b"], [20, 4], "cpu")
    a, b = t.slots("a", "cpu").tolist(), t.slots("b", "cpu").tolist()
    src, dst, starts, most = t.accept(["b", "a"], [4, 20], [[0, 1], [0, 3, 19]], "cpu")
    assert src.tolist() == [a[14 + 3], a[14 + 19]] and dst.tolist() == [a[15], a[16]] and starts.tolist() == [0, 0, 2] and most == 2
    assert starts.dtype == torch.int32 and src.dtype == torch.int64
    assert t.length("a") == 17 and t.length("b") == 5 and t.slots("a", "cpu").tolist() == a[:17] and t.free_pages == 8 - 2 - 1
    assert t.accept(["a"], [17], [[]], "cpu")[3] == 0 and t.length("a") == 0 and t.free_pages == 7
    assert t.accept([], [], [], "cpu")[2].tolist() == [0]
    assert b[:5] == t.slots("b", "cpu").tolist()


def test_accept_refuses_and_changes_nothing():
    t = table(a=20, b=20)
    for counts, kept in (([21], [[0]]), ([4], [[4]]), ([4], [[-1]]), ([4], [[2, 1]]), ([4], [[1, 1]]), ([-1], [[]])):
        with pytest.raises(ValueError, match="numbers kept"):
            t.accept(["a"], counts, kept, "cpu")
    for args in ((["a", "a"], [1, 1], [[], []]), (["a"], [1, 2], [[]]), (["a"], [1], [])):
        with pytest.raises(ValueError):
            t.accept(*args, "cpu")
    with pytest.raises(ValueError):
        t.accept(["b", "a"], [2, 4], [[0], [9]], "cpu")                    # the second is wrong: the first stays as it is
    assert t.length("a") == t.length("b") == 20 and t.free_pages == 4


def test_drafts_in_shared_pages_stay():
    t = table(a=20)
    t.extend(["a"], [20], "cpu")                                           # pages 0 (20 tokens before: 0, 1), drafts in 1 and 2
    t.fork(["a"], ["x"], "cpu")                                            # shares 0 and 1
    for kept in ([], [0, 2], [3], list(range(19, 20))):
        with pytest.raises(ValueError, match="shares"):
            t.accept(["a"], [20], [kept], "cpu")
    t.accept(["a"], [20], [list(range(20))], "cpu")                        # all of them: nothing is written
    t.accept(["x"], [8], [[2]], "cpu")                                     # in the page of its own
    assert t.length("x") == 33 and t.length("a") == 40
    t.accept(["a"], [8], [[]], "cpu")                                      # down to a full page: its next token takes a new one
    assert t.length("a") == 32 and len(t._pages["a"]) == 2
    t.remove("x")
    t.accept(["a"], [12], [[]], "cpu")                                     # its own again
    assert t.length("a") == 20


def test_compact():
    t = table(a=16, b=40, c=16)
    t.fork(["b"], ["x"], "cpu")
    t.remove("a")
    t.remove("b")
    held = {s: t._pages[s][:] for s in ("c", "x")}
    src, dst = t.compact("cpu")
    place = dict(zip(src.tolist(), dst.tolist()))
    assert set(src.tolist()).isdisjoint(dst.tolist()) and all(p >= 4 for p in src.tolist()) and all(p < 4 for p in dst.tolist())
    for s, pages in held.items():
        assert t._pages[s] == [place.get(p, p) for p in pages]
    assert t.free_pages == 4 and sorted(t._free) == [4, 5, 6, 7] and [o > 0 for o in t._owners] == [True] * 4 + [False] * 4
    assert t.compact("cpu")[0].shape == (0,)
    s = t.extend(["c"], [1], "cpu")
    assert s.item() == 4 * 16
    t = table(a=20)
    t.fork(["a"], ["x"], "cpu")
    t.remove("a")                                                          # a shared page moves once, for all
    t.add("z")
    t.extend(["z"], [16], "cpu")
    t.fork(["x"], ["y"], "cpu")
    t.remove("z")
    t.compact("cpu")
    assert t._pages["x"][0] == t._pages["y"][0] and t._owners[t._pages["x"][0]] == 2


def test_positions():
    t = table(a=20, b=3)
    p = t.positions(["b", "a"], [2, 3], "cpu")
    assert p.tolist() == [1, 2, 17, 18, 19] and p.dtype == torch.int32


# ------------------------------------------------------------------------------------------------ rotary tables
def test_turns():
    rot = Rotary(64, base=10.0, sections=(8, 24), restart=True, device="cpu")
    assert rot.axes == (0,) * 8 + (1,) * 24 and rot.n_axes == 2 and rot.frequencies[8] == 1.0 and rot.frequencies[9] == 10.0 ** (-2 / 48)
    for t, f in zip(rot.turns.tolist(), rot.frequencies):
        assert abs(t / 2.0 ** 64 - f / (2 * math.pi)) < 2.0 ** -50
    fast = Rotary(64, frequencies=[5.0, -1.0] + [0.0] * 30, device="cpu").turns.tolist()
    assert fast[0] < 0 and abs(fast[0] / 2.0 ** 64 + 1 - 5.0 / (2 * math.pi)) < 2.0 ** -50 and fast[1] < 0 and fast[2] == 0


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=80), dict(sections=(16, 15)), dict(sections=(32, 0)), dict(base=0.0),
                                dict(base=math.inf), dict(frequencies=[1.0]), dict(frequencies=[math.nan] * 32), dict(axes=[0] * 31), dict(axes=[-1] * 32),
                                dict(axes=[0] * 32, sections=(32,)), dict(axes=[0] * 32, restart=True)])
def test_rotary_refuses(kw):
    with pytest.raises(ValueError, match="VAR-Q"):
        Rotary(**{"head_dim": 64, "device": "cpu", **kw})


def test_cpu_tensors_are_refused():
    rot, x, p = Rotary(64, device="cpu"), torch.zeros(2, 1, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        rot.rotate(x, x, p)
    with pytest.raises(ValueError, match="norm"):
        rot.rotate(x, x, p, norm="max")
    with pytest.raises(RuntimeError, match="CUDA"):
        draft_tree(p, p, p, 1)
    with pytest.raises(TypeError, match="list"):
        from VAR_Q.rotary import _native
        _native().paged_copy_pages(None, p, p)
    assert copy_pages([], p, p) is None


# ------------------------------------------------------------------------------------------------ the C entries
def descriptors():
    cache = _cabi.Paged(256, 256, 256, 256, 4, 16, 2, 64, 8, 8)
    rot = _cabi.Rotary(256, 256, 256, 0, 0, 1, None, None, 0, 0, 0, 0, 4, 1, 64, 0, 0, 1e-6)
    t = _cabi.Tensor(256, _cabi.F16, 0, 0, 128, 64)
    return cache, rot, t


@pytest.mark.parametrize("field,value,rc,word", [
    ("rotary_dim", 8, -2, b"rotary_dim"), ("rotary_dim", 72, -2, b"rotary_dim"), ("rotary_dim", 80, -2, b"rotary_dim"), ("n_axes", 0, -1, b"axes"), ("pos_bytes", 2, -1, b"positions"), ("norm", 3, -1, b"norm"),
    ("turns", None, -1, b"null"), ("axis", None, -1, b"null"), ("positions", None, -1, b"null"), ("positions", 258, -1, b"misaligned"), ("turns", 260, -1, b"misaligned"),
    ("q_weight", 257, -1, b"misaligned")])
def test_c_entries_check_the_rotary_descriptor(field, value, rc, word):
    lib = _cabi.lib()
    cache, rot, t = descriptors()
    setattr(rot, field, value)
    assert lib.varq_rotate(rot, t, t, 1, 4, 2, 2, 64, t, t, None) == rc and word in lib.varq_last_error()
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, 256, 4, 2, 1e-12, t, None) == rc and word in lib.varq_last_error()


def test_more_refusals_and_empty_calls_of_rotations():
    lib = _cabi.lib()
    cache, rot, t = descriptors()
    f32, bf16 = (_cabi.Tensor(256, d, 0, 0, 128, 64) for d in (_cabi.F32, _cabi.BF16))
    assert lib.varq_rotate(rot, t, t, 0, 4, 2, 2, 64, t, t, None) == 0 and lib.varq_rotate(rot, t, t, 1, 4, 0, 0, 64, t, t, None) == 0
    assert lib.varq_rotate(rot, t, t, 1, 4, 2, 2, 96, t, t, None) == -2 and b"head_dim" in lib.varq_last_error()
    assert lib.varq_rotate(rot, t, f32, 1, 4, 2, 2, 64, t, t, None) == -1 and lib.varq_rotate(rot, t, t, 1, 4, 2, 2, 64, bf16, bf16, None) == -1
    assert lib.varq_rotate(rot, t, t, 1, 4, 2, 2, 64, t, f32, None) == -1
    assert lib.varq_rotate(rot, t, t, -1, 4, 2, 2, 64, t, t, None) == -1 and lib.varq_rotate(rot, t, t, 1, 4, -1, 2, 64, t, t, None) == -1
    assert lib.varq_rotate(rot, t, t, 1 << 15, 1 << 15, 2, 2, 64, t, t, None) == -2 and b"2^31" in lib.varq_last_error()
    assert lib.varq_rotate(None, t, t, 1, 4, 2, 2, 64, t, t, None) == -1 and lib.varq_rotate(rot, None, t, 1, 4, 2, 2, 64, t, t, None) == -1
    rot.norm, rot.eps = 2, 0.0
    assert lib.varq_rotate(rot, t, t, 1, 4, 2, 2, 64, t, t, None) == -1 and b"eps" in lib.varq_last_error()
    cache, rot, t = descriptors()
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, 256, 0, 2, 1e-12, t, None) == 0
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, 256, -1, 2, 1e-12, t, None) == -1
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, 256, 1 << 29, 2, 1e-12, t, None) == -2
    assert lib.varq_paged_append_rotated(cache, rot, t, t, bf16, 256, 4, 2, 1e-12, t, None) == -1
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, 256, 4, 2, 1e-12, f32, None) == -1
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, None, 4, 2, 1e-12, t, None) == -1
    assert lib.varq_paged_append_rotated(cache, rot, t, t, t, 256, 4, 2, 0.0, t, None) == -1 and b"eps" in lib.varq_last_error()
    assert lib.varq_paged_append_rotated(None, rot, t, t, t, 256, 4, 2, 1e-12, t, None) == -1


def test_refusals_and_empty_calls_of_copies_and_trees():
    lib = _cabi.lib()
    two = (_cabi.Paged * 2)(descriptors()[0], descriptors()[0])
    assert lib.varq_paged_move_tokens(two, 2, 256, 256, 3, 256, 1, 0, None) == -1 and b"0 and 1 are one" in lib.varq_last_error()
    two[1].k_codes = two[0].k_codes + 256
    assert lib.varq_paged_copy_pages(two, 2, 256, 256, 0, None) == 0 and lib.varq_paged_copy_pages(None, 0, 256, 256, 3, None) == 0
    assert lib.varq_paged_copy_pages(two, -1, 256, 256, 3, None) == -1 and lib.varq_paged_copy_pages(None, 2, 256, 256, 3, None) == -1
    assert lib.varq_paged_copy_pages(two, 2, None, 256, 3, None) == -1 and lib.varq_paged_copy_pages(two, 2, 256, 260, 3, None) == -1
    assert lib.varq_paged_copy_pages(two, 2, 256, 256, -3, None) == -1
    assert lib.varq_paged_move_tokens(two, 2, 256, 256, 0, 256, 1, 0, None) == 0 and lib.varq_paged_move_tokens(two, 2, 256, 256, 3, 256, 0, 0, None) == 0
    assert lib.varq_paged_move_tokens(two, 2, 256, 256, 3, None, 1, 0, None) == -1 and lib.varq_paged_move_tokens(two, 2, 256, 256, 3, 257, 1, 0, None) == -1
    assert lib.varq_paged_move_tokens(two, 2, 256, 256, 3, 256, -1, 0, None) == -1 and lib.varq_paged_move_tokens(two, 2, 256, 256, 3, 256, 1, -1, None) == -1
    two[1].page_size = 32
    for rc in (lib.varq_paged_copy_pages(two, 2, 256, 256, 3, None), lib.varq_paged_move_tokens(two, 2, 256, 256, 3, 256, 1, 0, None)):
        assert rc == -1 and b"16 and 32" in lib.varq_last_error()
    two[1].page_size, two[1].k_bits = 16, 3
    assert lib.varq_paged_copy_pages(two, 2, 256, 256, 0, None) == -1 and b"bits" in lib.varq_last_error()
    assert lib.varq_paged_tree(256, 256, 256, 1, 0, 4, 1, 256, 256, None) == 0
    assert lib.varq_paged_tree(256, 256, 256, 1, 4, 33, 1, 256, 256, None) == -1 and b"words" in lib.varq_last_error()
    assert lib.varq_paged_tree(None, 256, 256, 1, 4, 4, 1, 256, 256, None) == -1 and lib.varq_paged_tree(256, None, 256, 1, 4, 4, 1, 256, 256, None) == -1
    assert lib.varq_paged_tree(256, 256, 256, -1, 4, 4, 1, 256, 256, None) == -1 and lib.varq_paged_tree(256, 256, 258, 1, 4, 4, 1, 256, 256, None) == -1
    cache, _, t = descriptors()
    for tree, words, field, value, word in ((256, 1, "causal", 0, b"causal"), (256, 0, "window", 0, b"words"), (256, 1, "window", 2, b"window"),
                                            (258, 1, "window", 0, b"misaligned"), (None, 1, "window", 0, b"null")):
        batch = _cabi.PagedBatch(256, 256, 256, 4, 6, 4, 2, 4, 3, 64, 1, 0, 0, 0.125)
        setattr(batch, field, value)
        assert lib.varq_paged_attn_tree(cache, batch, tree, words, t, t, None, None, 0, None) == -1 and word in lib.varq_last_error()
    # the descriptor of a batch is what it was: who calls varq_paged_attn with it needs no new one
    assert ctypes.sizeof(_cabi.PagedBatch) == 80
