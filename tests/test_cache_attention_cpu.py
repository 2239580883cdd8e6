"""The entry points over a key-value cache without a GPU: what they refuse, before any device work. The views lie over
addresses that are never touched: a call that passes every check ends at the missing device, with another code."""
import pytest


def at(F, shape, dtype, stride=None, address=1 << 20, room=1 << 40):
    return F.Tensor.from_device_ptr(address, shape, dtype, stride=stride, numel=room)


def operands(F, dt, N=2, H=4, Hk=2, L=1, S=10, D=64, P=6):
    t = {"q": at(F, (N, H, L, D), dt), "k": at(F, (N, Hk, S, D), dt), "v": at(F, (N, Hk, S, D), dt), "out": at(F, (N, H, L, D), dt, address=1 << 28),
         "pk": at(F, (1, Hk, P, D), dt), "pv": at(F, (1, Hk, P, D), dt), "lens": at(F, (N,), F.DType.INT32),
         "w": at(F, (N, Hk, S), F.DType.FLOAT), "wo": at(F, (N, Hk, S), F.DType.FLOAT, address=1 << 30)}
    return t


class NoDevice:
    def __init__(self, F):
        self.F = F

    def refused(self, call, *args):
        code = call(*[a.raw() if hasattr(a, "raw") else a for a in args])
        assert code != self.F.FL_OK
        return code == self.F.FL_ERROR_INVALID_ARG, self.F.lib().fl_get_last_error_message().decode()


@pytest.fixture()
def no_device(flint):
    import ctypes
    import torch
    if torch.cuda.is_available():
        pytest.skip("a valid call would run")
    return NoDevice(flint), ctypes.c_void_p(1)  # (operators cannot be made without a device: what is not null stands for them)


def test_what_attention_refuses(flint, no_device):
    F, (N, ops) = flint, no_device
    L = F.lib()
    bf, half = F.DType.BFLOAT16, F.DType.FLOAT16
    t = operands(F, bf)
    window = lambda **c: N.refused(L.fl_attention_window, ops, *[{**t, **c}[n] for n in ("q", "k", "v", "lens")], c.get("window", 5),  # noqa: E731
                                   c.get("sinks", 0), {**t, **c}["out"])
    assert not window()[0]      # the operands are fine: only the device is missing
    assert not window(lens=None)[0]
    bad = [
        (dict(window=0), "a window of 0"), (dict(window=-3), "a window of -3"), (dict(sinks=-1), "first keys"),
        (dict(k=at(F, (2, 3, 10, 64), bf), v=at(F, (2, 3, 10, 64), bf)), "multiple of the key-value heads"),
        (dict(k=at(F, (2, 2, 0, 64), bf), v=at(F, (2, 2, 0, 64), bf)), "no keys"),
        (dict(v=at(F, (2, 2, 9, 64), bf)), "disagree"), (dict(out=at(F, (2, 4, 2, 64), bf)), "out is not of q's shape"),
        (dict(k=at(F, (2, 2, 10, 64), half)), "one type"), (dict(q=at(F, (2, 4, 64), bf)), "four-dimensional"),
        (dict(q=at(F, (2, 4, 1, 96), bf), out=at(F, (2, 4, 1, 96), bf), k=at(F, (2, 2, 10, 96), bf), v=at(F, (2, 2, 10, 96), bf)), "64 or 128"),
        (dict(k=at(F, (2, 2, 10, 64), bf, (1280, 640, 64, 2))), "k's last dimension"),
        (dict(k=at(F, (2, 2, 10, 64), bf, (0, 640, 64, 1))), "stride of 0"), (dict(out=at(F, (2, 4, 1, 64), bf, (0, 64, 64, 1))), "stride of 0"),
        (dict(v=at(F, (2, 2, 10, 64), bf, (1300, 650, 65, 1))), "multiple of 8"), (dict(q=at(F, (2, 4, 1, 64), bf, address=(1 << 20) + 2)), "16-byte"),
        (dict(out=t["q"]), "out shares elements with q"), (dict(out=at(F, (2, 4, 1, 64), bf, address=(1 << 20) + 2304)), "shares elements with k"),
        (dict(lens=at(F, (3,), F.DType.INT32)), "kv_lens"), (dict(lens=at(F, (2,), F.DType.LONG)), "kv_lens"),
        (dict(lens=at(F, (2,), F.DType.INT32, (2,))), "kv_lens"),
    ]
    for change, words in bad:
        refusal, message = window(**change)
        assert refusal and words in message, (change.keys(), message)
    assert window(q=at(F, (2, 4, 1, 64), bf, (0, 64, 64, 1)))[0]
    assert N.refused(L.fl_attention_window, None, t["q"], t["k"], t["v"], None, 5, 0, t["out"])[0]

    prefix = lambda **c: N.refused(L.fl_attention_shared_prefix, ops, *[{**t, **c}[n] for n in ("q", "pk", "pv", "k", "v", "lens", "out")])  # noqa: E731
    assert not prefix()[0]
    between = dict(q=at(F, (2, 4, 1, 64), bf, (1024, 128, 128, 1)), out=at(F, (2, 4, 1, 64), bf, (1024, 128, 128, 1), (1 << 20) + 128))
    far = dict(k=at(F, (2, 2, 10, 64), bf, address=1 << 29), v=at(F, (2, 2, 10, 64), bf, address=1 << 29))
    assert not window(**between, **far)[0]  # q and out take turns in memory
    for change, words in [(dict(out=at(F, (2, 4, 1, 64), bf, address=(1 << 20) + 512), **far), "shares elements with q"), (dict(out=at(F, (2, 4, 1, 64), bf), **far, q=at(F, (2, 4, 1, 64), bf, address=1 << 27)), "prefix"),
                          (dict(pk=at(F, (2, 2, 6, 64), bf)), "(1, kv_heads, length, head_dim)"), (dict(pv=at(F, (1, 2, 7, 64), bf)), "disagree"),
                          (dict(pk=at(F, (1, 2, 0, 64), bf), pv=at(F, (1, 2, 0, 64), bf)), "empty prefix"), (dict(pk=at(F, (1, 2, 6, 64), half)), "type"),
                          (dict(pk=at(F, (1, 2, 6, 64), bf, (768, 384, 0, 1))), "stride of 0"), (dict(pv=at(F, (1, 2, 6, 64), bf, address=(1 << 20) + 8)), "16-byte")]:
        refusal, message = prefix(**change)
        assert refusal and words in message, (change.keys(), message)

    weights = lambda **c: N.refused(L.fl_attention_weights, ops, *[{**t, **c}[n] for n in ("q", "k", "v", "lens", "w", "wo", "out")])  # noqa: E731
    assert not weights()[0]
    assert not weights(wo=t["w"])[0]
    for change, words in [(dict(w=at(F, (2, 2, 9), F.DType.FLOAT)), "weights"), (dict(wo=at(F, (2, 2, 10), bf)), "weights_out"),
                          (dict(wo=at(F, (2, 2, 10), F.DType.FLOAT, (40, 20, 2), 1 << 30)), "contiguous"),
                          (dict(wo=at(F, (2, 2, 10), F.DType.FLOAT, (0, 10, 1), 1 << 30)), "stride of 0"),
                          (dict(wo=at(F, (2, 2, 10), F.DType.FLOAT, address=(1 << 20) + 4)), "overlap"),
                          (dict(q=at(F, (2, 4, 0, 64), bf), out=at(F, (2, 4, 0, 64), bf)), "no queries")]:
        refusal, message = weights(**change)
        assert refusal and words in message, (change.keys(), message)


def test_what_eviction_refuses(flint, no_device):
    F, (N, ops) = flint, no_device
    L = F.lib()
    bf, fl = F.DType.BFLOAT16, F.DType.FLOAT
    far = lambda i: (i + 2) << 32  # noqa: E731
    t = {"k": at(F, (2, 2, 10, 24), bf), "v": at(F, (2, 2, 10, 24), bf), "w": at(F, (2, 2, 10), fl), "lens": at(F, (2,), F.DType.INT32, address=far(8)),
         "ko": at(F, (2, 2, 6, 24), bf, address=far(0)), "vo": at(F, (2, 2, 6, 24), bf, address=far(1)), "wo": at(F, (2, 2, 6), fl, address=far(2)),
         "lo": at(F, (2,), F.DType.INT32, address=far(3)), "kept": at(F, (2, 2, 5), F.DType.INT32, address=far(4))}

    def evict(keep=5, recent=2, **c):
        u = {**t, **c}
        return N.refused(L.fl_cache_evict, ops, u["k"], u["v"], u["w"], u["lens"], keep, recent, u["ko"], u["vo"], u["wo"], u["lo"], u["kept"])

    assert not evict()[0] and not evict(kept=None)[0] and not evict(lens=None, lo=None)[0] and not evict(lo=t["lens"])[0]
    for change, words in [
            (dict(keep=0), "0 keys to keep"), (dict(keep=7), "room for 6"), (dict(recent=6), "recent"), (dict(recent=-1), "recent"),
            (dict(v=at(F, (2, 2, 9, 24), bf)), "disagree"), (dict(vo=at(F, (2, 2, 7, 24), bf, address=far(1))), "disagree"),
            (dict(ko=at(F, (2, 2, 6, 24), F.DType.FLOAT16, address=far(0))), "one type"), (dict(w=at(F, (2, 2, 6), fl)), "weights"),
            (dict(wo=at(F, (2, 2, 10), fl, address=far(2))), "weights_out"), (dict(lo=None), "lens_out"), (dict(lens=at(F, (1,), F.DType.INT32)), "kv_lens"),
            (dict(kept=at(F, (2, 2, 6), F.DType.INT32, address=far(4))), "kept"), (dict(ko=at(F, (2, 2, 6, 24), bf, address=(1 << 20) + 16)), "overlaps k, v or weights"),
            (dict(lo=at(F, (2,), F.DType.INT32, address=far(8) + 4)), "lens_out overlaps kv_lens"),
            (dict(lo=at(F, (2,), F.DType.INT32, address=far(2) + 16)), "two outputs"),
            (dict(vo=t["ko"]), "two outputs"), (dict(ko=at(F, (2, 2, 6, 24), bf, (0, 144, 24, 1), far(0))), "stride of 0"),
            (dict(k=at(F, (2, 2, 10, 24), bf, (480, 240, 24, 1), (1 << 20) + 2)), "16-byte")]:
        refusal, message = evict(**change)
        assert refusal and words in message, (change.keys(), message)
    assert evict(k=at(F, (2, 2, 10, 20), bf), v=at(F, (2, 2, 10, 20), bf), ko=at(F, (2, 2, 6, 20), bf, address=far(0)), vo=at(F, (2, 2, 6, 20), bf, address=far(1)))[0]
    assert not evict(k=at(F, (2, 2, 10, 24), bf, (0, 0, 24, 1)))[0]  # read with their true strides: inputs may repeat


def test_outputs_that_take_turns_in_memory(flint, no_device):
    """A cache that keeps keys and values side by side, (N, S, 2, kv_heads, D), is taken for both; one element in common is not."""
    F, (N, ops) = flint, no_device
    L = F.lib()
    bf, fl = F.DType.BFLOAT16, F.DType.FLOAT
    far = lambda i: (i + 2) << 32  # noqa: E731
    side = lambda address, i, rows=6: at(F, (2, 2, rows, 24), bf, (2 * 48 * rows, 24, 96, 1), address + int(96 * i))  # noqa: E731  (keys 0, values 1)
    t = {"k": at(F, (2, 2, 10, 24), bf), "v": at(F, (2, 2, 10, 24), bf), "w": at(F, (2, 2, 10), fl), "lens": at(F, (2,), F.DType.INT32, address=far(8)),
         "ko": at(F, (2, 2, 6, 24), bf, address=far(0)), "vo": at(F, (2, 2, 6, 24), bf, address=far(1)), "wo": at(F, (2, 2, 6), fl, address=far(2)),
         "lo": at(F, (2,), F.DType.INT32, address=far(3)), "kept": at(F, (2, 2, 5), F.DType.INT32, address=far(4))}

    def evict(**c):
        u = {**t, **c}
        return N.refused(L.fl_cache_evict, ops, u["k"], u["v"], u["w"], u["lens"], 5, 2, u["ko"], u["vo"], u["wo"], u["lo"], u["kept"])

    assert not evict(ko=side(far(0), 0), vo=side(far(0), 1))[0]
    refusal, message = evict(ko=side(far(0), 0), vo=side(far(0), 0.5))
    assert refusal and "two outputs" in message
    # Both caches in one allocation, sequence by sequence.
    old = lambda i: at(F, (2, 2, 10, 24), bf, (4096, 240, 24, 1), far(0) + 1024 * i)  # noqa: E731
    new = lambda i: at(F, (2, 2, 6, 24), bf, (4096, 144, 24, 1), far(0) + 2048 + 1024 * i)  # noqa: E731
    assert not evict(k=old(0), v=old(1), ko=new(0), vo=new(1))[0]
    refusal, message = evict(k=old(0), v=old(1), ko=new(0), vo=new(-1))
    assert refusal and "overlaps k, v or weights" in message
    # Weights of two steps that take turns, head by head.
    step = lambda i: at(F, (2, 2, 10), fl, (40, 20, 1), far(5) + i)  # noqa: E731
    q = operands(F, bf)
    weights = lambda w, wo: N.refused(L.fl_attention_weights, ops, q["q"], q["k"], q["v"], q["lens"], w, wo, q["out"])  # noqa: E731
    assert not weights(step(0), step(40))[0] and not weights(step(40), step(40))[0]
    refusal, message = weights(step(0), step(36))
    assert refusal and "overlap" in message
    one = at(F, (1, 2, 10), fl, (20, 10, 1), far(5)), at(F, (1, 2, 10), fl, (0, 10, 1), far(5))  # the same, a stride that is never used apart
    single = operands(F, bf, N=1)
    assert not N.refused(L.fl_attention_weights, ops, single["q"], single["k"], single["v"], None, *one, single["out"])[0]


def test_an_output_that_shares_elements_with_neither_view_whole(flint, no_device):
    """Strided views that meet in the middle alone: the one's ends lie between the other's elements."""
    F, (N, ops) = flint, no_device
    bf = F.DType.BFLOAT16
    t = operands(F, bf, N=3, H=2, Hk=2)
    k = at(F, (3, 2, 10, 64), bf, (4096, 1024, 64, 1), 1 << 24)
    for delta, shares in ((0, True), (128, True), (1280, False), (3 * 4096 * 2, False), (-2 * 4096 * 2 + 128, True), (-2 * 4096 * 2 - 128, False)):
        out = at(F, (3, 2, 1, 64), bf, (4096, 1024, 64, 1), (1 << 24) + delta)
        refusal, message = N.refused(F.lib().fl_attention_window, ops, t["q"], k, t["v"], None, 5, 0, out)
        assert refusal == shares and (not shares or "shares elements with k" in message), (delta, message)


def test_shared_elements_against_sets_of_them(flint, no_device):
    """Random layouts: refused exactly where a set of the one view's elements meets a set of the other's."""
    import random
    import numpy as np
    F, (N, ops) = flint, no_device
    bf, D, rng = F.DType.BFLOAT16, 64, random.Random(4)

    def layout(shape, gaps):
        order, strides, step = [0, 1, 2], [0, 0, 0], D
        rng.shuffle(order)
        for d in order:
            strides[d] = step + rng.choice(gaps)
            step = strides[d] * shape[d]
        return strides

    def elements(shape, strides, start):
        grid = sum(np.arange(n).reshape([-1 if i == j else 1 for j in range(4)]) * s for i, (n, s) in enumerate(zip((*shape, D), (*strides, 1))))
        return set((grid + start).ravel().tolist())

    seen = {True: 0, False: 0}
    for _ in range(300):
        n, hk, l, s = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 5)
        out, keys = (n, hk, l), (n, hk, s)
        so, sk = layout(out, [0, 64, 256, 960]), layout(keys, [0, 64, 64, 192, 1032]) if rng.random() < 0.7 else [8 * rng.randint(1, 60) for _ in range(3)]
        start = 1 << 20
        delta = 8 * rng.randint(-200, 600)
        t = {"q": at(F, (*out, D), bf, address=1 << 40), "v": at(F, (*keys, D), bf, address=1 << 41),
             "k": at(F, (*keys, D), bf, (*sk, 1), 2 * start), "out": at(F, (*out, D), bf, (*so, 1), 2 * (start + delta))}
        refusal, message = N.refused(F.lib().fl_attention_window, ops, t["q"], t["k"], t["v"], None, 5, 0, t["out"])
        shares = not elements(keys, sk, start).isdisjoint(elements(out, so, start + delta))
        assert refusal == shares and (not shares or "shares elements with k" in message), (out, so, keys, sk, delta, message)
        seen[shares] += 1
    assert min(seen.values()) > 50


def test_every_output_is_compared_with_every_input(flint, no_device):
    F, (N, ops) = flint, no_device
    L = F.lib()
    bf, fl, i32 = F.DType.BFLOAT16, F.DType.FLOAT, F.DType.INT32
    far = lambda i: (i + 2) << 32  # noqa: E731
    q = {name: at(F, (2, h, n, 64), bf, address=far(i)) for i, (name, h, n) in enumerate((("q", 4, 1), ("k", 2, 10), ("v", 2, 10), ("out", 4, 1)))}
    q.update(lens=at(F, (2,), i32, address=far(4)), w=at(F, (2, 2, 10), fl, address=far(5)), wo=at(F, (2, 2, 10), fl, address=far(6)))
    over = lambda x, shift=16: (at(F, (2, 4, 1, 64), bf, address=x + shift))  # noqa: E731
    weights = lambda **c: N.refused(L.fl_attention_weights, ops, *[{**q, **c}[n] for n in ("q", "k", "v", "lens", "w", "wo", "out")])  # noqa: E731
    window = lambda **c: N.refused(L.fl_attention_window, ops, *[{**q, **c}[n] for n in ("q", "k", "v", "lens")], 5, 0, {**q, **c}["out"])  # noqa: E731
    assert not weights()[0] and not window()[0]
    refusal, message = window(lens=at(F, (2,), i32, address=far(3) + 16))
    assert refusal and "out shares elements with kv_lens" in message
    refusal, message = weights(out=over(far(5)))
    assert refusal and "out shares elements with weights" in message
    for i, name in enumerate(("q", "k", "v", "out", "kv_lens")):
        refusal, message = weights(wo=at(F, (2, 2, 10), fl, address=far(i) + 4))
        assert refusal and f"weights_out shares elements with {name}" in message, (name, message)
    assert not weights(lens=None, wo=at(F, (2, 2, 10), fl, address=far(4)))[0]
    t = {"k": at(F, (2, 2, 10, 24), bf), "v": at(F, (2, 2, 10, 24), bf), "w": at(F, (2, 2, 10), fl), "lens": at(F, (2,), i32, address=far(8) + 16),
         "ko": at(F, (2, 2, 6, 24), bf, address=far(0)), "vo": at(F, (2, 2, 6, 24), bf, address=far(1)), "wo": at(F, (2, 2, 6), fl, address=far(2)),
         "lo": at(F, (2,), i32, address=far(3)), "kept": at(F, (2, 2, 5), i32, address=far(4))}

    def evict(**c):
        u = {**t, **c}
        return N.refused(L.fl_cache_evict, ops, u["k"], u["v"], u["w"], u["lens"], 5, 2, u["ko"], u["vo"], u["wo"], u["lo"], u["kept"])

    for lo in (t["lo"], t["lens"]):
        assert not evict(lo=lo)[0]
        for name, view in (("ko", at(F, (2, 2, 6, 24), bf, address=far(8))), ("vo", at(F, (2, 2, 6, 24), bf, address=far(8))),
                           ("wo", at(F, (2, 2, 6), fl, address=far(8))), ("kept", at(F, (2, 2, 5), i32, address=far(8)))):
            refusal, message = evict(lo=lo, **{name: view})
            assert refusal and "an output overlaps kv_lens" in message, (name, message)


def test_outputs_whose_own_elements_meet(flint, no_device):
    """Strides that lead to one place by two ways are refused in what is written, taken in what is read."""
    F, (N, ops) = flint, no_device
    L = F.lib()
    bf, fl = F.DType.BFLOAT16, F.DType.FLOAT
    far = lambda i: (i + 2) << 32  # noqa: E731
    t = operands(F, bf, N=3, H=4, Hk=2, L=5)
    shape = (3, 4, 5, 64)
    window = lambda out, k=t["k"]: N.refused(L.fl_attention_window, ops, t["q"], k, t["v"], None, 5, 0, out)  # noqa: E731
    for strides, meets in [((1280, 320, 64, 1), False), ((1280, 64, 256, 1), False), ((64, 192, 768, 1), False), ((1280, 320, 56, 1), True),
                           ((1280, 256, 64, 1), True), ((1280, 64, 64, 1), True), ((128, 1024, 192, 1), True), ((128, 2048, 320, 1), False),
                           ((3 * 64, 3 * 2 * 5 * 64, 2 * 64, 1), True)]:
        refusal, message = window(at(F, shape, bf, strides, far(3)))
        assert refusal == meets and (not meets or "two elements in one place" in message), (strides, message)
    assert not window(at(F, shape, bf, address=far(3)), at(F, (3, 2, 10, 64), bf, (640, 320, 8, 1)))[0]
    w = lambda strides: at(F, (3, 2, 10), fl, strides, far(5))  # noqa: E731
    for strides, meets in [((20, 10, 1), False), ((10, 30, 1), False), ((10, 10, 1), True), ((20, 9, 1), True)]:
        refusal, message = N.refused(L.fl_attention_weights, ops, t["q"], t["k"], t["v"], None, at(F, (3, 2, 10), fl, address=far(6)), w(strides), at(F, shape, bf, address=far(3)))
        assert refusal == meets and (not meets or "two elements in one place" in message), (strides, message)
    e = {"k": at(F, (2, 2, 10, 24), bf), "v": at(F, (2, 2, 10, 24), bf), "w": at(F, (2, 2, 10), fl), "ko": at(F, (2, 2, 6, 24), bf, address=far(0)),
         "vo": at(F, (2, 2, 6, 24), bf, address=far(1)), "wo": at(F, (2, 2, 6), fl, address=far(2))}
    for name, view in [("ko", at(F, (2, 2, 6, 24), bf, (288, 136, 24, 1), far(0))), ("vo", at(F, (2, 2, 6, 24), bf, (288, 144, 16, 1), far(1))),
                       ("wo", at(F, (2, 2, 6), fl, (12, 5, 1), far(2)))]:
        u = {**e, name: view}
        refusal, message = N.refused(L.fl_cache_evict, ops, u["k"], u["v"], u["w"], None, 5, 2, u["ko"], u["vo"], u["wo"], None, None)
        assert refusal and "two elements in one place" in message, (name, message)
    assert not N.refused(L.fl_cache_evict, ops, e["k"], e["v"], e["w"], None, 5, 2, e["ko"], e["vo"], e["wo"], None, None)[0]


def test_more_positions_than_32_bits_hold(flint, no_device):
    """A query's position less a window of 2^30 keys has to be an int: 2^30 queries at most, and as many keys."""
    F, (N, ops) = flint, no_device
    bf = F.DType.BFLOAT16
    kv = at(F, (1, 1, 1 << 30, 64), bf, (64, 64, 8, 1))
    for queries in (1 << 30, (1 << 30) + 1):
        q, out = (at(F, (1, 1, queries, 64), bf, (64, 64, step, 1), address=(i + 1) << 42) for i, step in enumerate((8, 64)))
        refusal, message = N.refused(F.lib().fl_attention_window, ops, q, kv, kv, None, 1 << 30, 0, out)
        assert refusal == (queries > 1 << 30) and (not refusal or "more than 2^30 queries" in message), message
