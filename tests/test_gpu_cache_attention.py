"""GPU parity of the entry points over a decoder's key-value cache with a plain float64 implementation.

Tolerance of an output element, u half a step of the type (2^-8 bfloat16, 2^-11 half), n keys seen, A the sum of
weight x |value| over them, B the largest sum of |q k| / sqrt(D) behind a score, by arithmetic:
  u |want|                the one rounding at the end;
  u A                     probabilities rounded to 16 bits before the second product (where they are);
  2 (D + 4) 2^-23 B A     the scores' float sums: D products, each addition off by at most one part in 2^23 (tensor
                          cores truncate) of the sum of magnitudes, in a weight's numerator and in its denominator;
  (2^-12 + n 2^-23) A     exponentials (a cubic good to 7.5e-5 in numerator and denominator) and the sums over keys.
These are sums of the worst; over a whole result, where roundings are spread evenly, fl_attention's bound holds too: a
relative L2 error of at most 5e-3.
A key's weight W, added up over R queries: 2 (D + 4) 2^-23 B + 2^-20 + 2^-13 + (n + R) 2^-23 of it (exponentials by the
hardware's function, 2^-22, but for the rows' sums, which may hold the cubic's 7.5e-5 < 2^-13), and 2^-23 of the total
for the additions to what was there."""
import numpy as np
import pytest

import cache_oracle as C

pytestmark = pytest.mark.gpu


def dev(F, a, dtype):
    return F.Tensor.from_numpy(a, dtype, F.Device.CUDA)


def types(F, is_bf16):
    return F.DType.BFLOAT16 if is_bf16 else F.DType.FLOAT16


class Cache:
    """Random operands, on the host as values and on the device as views, head-major or token-major in memory."""

    def __init__(self, F, O, seed, N, H, Hk, L, S, D, is_bf16, lens=None, tokens=False, P=0, spread=1.0):
        rng = np.random.default_rng(seed)
        self.F, self.O, self.is_bf16, self.tokens = F, O, is_bf16, tokens
        self.shape = (N, H, Hk, L, S, D)
        self.bits = {"q": self.draw(rng, N, H, L, D, spread), "k": self.draw(rng, N, Hk, S, D, spread), "v": self.draw(rng, N, Hk, S, D)}
        if P:
            self.bits["prefix_k"], self.bits["prefix_v"] = self.draw(rng, 1, Hk, P, D, spread), self.draw(rng, 1, Hk, P, D)
        self.lens = None if lens is None else np.asarray(lens, np.int32)

    def draw(self, rng, n, h, l, d, spread=1.0):
        return self.O.narrow((rng.standard_normal((n, h, l, d)) * spread).astype(np.float32), self.is_bf16)

    def value(self, name):
        return self.O.widen(self.bits[name], self.is_bf16).astype(np.float64)

    def view(self, a):
        dt = types(self.F, self.is_bf16)
        if not self.tokens:
            return dev(self.F, a, dt)
        n, h, l, d = a.shape
        store = dev(self.F, np.ascontiguousarray(a.transpose(0, 2, 1, 3)), dt)
        return store.view_as((n, h, l, d), (l * h * d, d, h * d, 1))

    def device(self):
        t = {name: self.view(a) for name, a in self.bits.items()}
        t["lens"] = None if self.lens is None else dev(self.F, self.lens, self.F.DType.INT32)
        n, h, hk, l, s, d = self.shape
        t["out"] = self.view(np.full((n, h, l, d), 0x7FC0 if self.is_bf16 else 0x7E00, np.uint16))  # NaN: every element is written
        return t

    def read(self, t):
        """The values of a (N, heads, length, D) view made by view()."""
        if self.tokens:
            n, h, l, d = t.shape
            return self.O.widen(t._keepalive.numpy(), self.is_bf16).transpose(0, 2, 1, 3).astype(np.float64)
        return self.O.widen(t.numpy(), self.is_bf16).astype(np.float64)


def check_out(got, want, size, score, keys, is_bf16, what):
    D = got.shape[-1]
    u = 2.0 ** (-8 if is_bf16 else -11)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    tol = u * np.abs(want) + (u + 2 * (D + 4) * 2.0 ** -23 * score + 2.0 ** -12 + keys * 2.0 ** -23) * size + (2.0 ** -24 if not is_bf16 else 0.0)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    with np.errstate(invalid="ignore"):
        off = (np.abs(got - want) / np.maximum(tol, 1e-30))[fine]
    assert off.size == 0 or off.max() <= 1.0, f"{what}: {off.max():.2f} of the tolerance"
    assert np.linalg.norm(got[fine] - want[fine]) <= 5e-3 * np.linalg.norm(want[fine]), f"{what}: relative L2"


WINDOW = [
    # N, H, Hk, L, S, D, window, sinks, lens
    (1, 1, 1, 1, 1, 64, 1, 0, None),
    (1, 8, 2, 1, 77, 64, 64, 4, None),
    (3, 7, 1, 1, 300, 128, 100, 3, [300, 0, 57]),          # a sequence without keys; an odd group
    (2, 32, 1, 1, 513, 128, 513, 0, [513, 200]),           # two tiles of query heads
    (2, 4, 4, 1, 5000, 128, 4096, 16, [5000, 4999]),       # many splits
    (1, 4, 2, 5, 900, 64, 33, 7, [871]),                   # a few tokens under a short window
    (2, 6, 2, 37, 333, 128, 20, 130, [333, 20]),           # sinks wider than the window; queries before every key
    (2, 3, 1, 130, 100, 64, 1000, 0, None),                # more queries than keys
    (1, 4, 1, 257, 1025, 128, 128, 1, None),
    (1, 2, 2, 600, 600, 64, 1, 0, None),                   # every query sees itself alone
    (2, 4, 2, 300, 700, 128, 250, 40, [700, 511]),
    (1, 3, 3, 1100, 1100, 128, 300, 4, [1093]),
    (1, 100, 1, 2, 300, 128, 77, 9, [291]),                # a tile of one query's 100 heads
    (1, 150, 1, 3, 200, 64, 60, 5, [170]),                 # more heads than a tile holds
    (3, 10, 2, 60, 70, 128, 9, 33, [70, 40, 0]),           # sinks beyond the window's start
    (2, 4, 4, 40, 9000, 64, 5000, 300, [9000, 8000]),      # few units whose blocks are divided; sinks over whole blocks
]


@pytest.mark.parametrize("N,H,Hk,L,S,D,window,sinks,lens", WINDOW)
@pytest.mark.parametrize("is_bf16,tokens", [(True, False), (False, True)])
def test_window(flint, oracle, N, H, Hk, L, S, D, window, sinks, lens, is_bf16, tokens):
    c = Cache(flint, oracle, 11 + L + S + H, N, H, Hk, L, S, D, is_bf16, lens, tokens)
    t = c.device()
    flint.attention_window(t["q"], t["k"], t["v"], window, sinks, t["lens"], t["out"])
    got = c.read(t["out"])
    flint.synchronize()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), lens, window, sinks)
    check_out(got, want, size, score, min(S, window + sinks), is_bf16, "window")
    if lens is not None:
        for n, length in enumerate(lens):
            if length < L:
                assert not got[n, :, :L - length].any()  # queries before every key


PREFIX = [
    # N, H, Hk, L, S, D, P, lens
    (1, 1, 1, 1, 1, 64, 1, None),
    (3, 8, 1, 1, 40, 64, 257, [40, 0, 13]),
    (9, 14, 2, 1, 65, 128, 1000, [65, 1, 2, 64, 33, 0, 17, 16, 5]),
    (5, 4, 2, 3, 100, 128, 130, [100, 2, 1, 0, 50]),     # queries that see the prefix alone
    (40, 8, 1, 1, 20, 128, 700, None),                   # more rows than a tile of the tensor cores
    (2, 4, 4, 200, 260, 64, 300, [260, 150]),
    (3, 4, 1, 129, 140, 128, 513, [140, 129, 60]),
    (1, 2, 1, 1, 30, 128, 5000, None),
    (30, 3, 1, 2, 50, 64, 1300, None),                   # 21 sequences of six rows to a tile
    (2, 150, 1, 1, 33, 64, 290, [33, 2]),                # more heads than a tile holds
    (2, 2, 1, 150, 200, 128, 3000, [200, 30]),           # few units whose walk over prefix and own keys is divided
]


@pytest.mark.parametrize("N,H,Hk,L,S,D,P,lens", PREFIX)
@pytest.mark.parametrize("is_bf16,tokens", [(True, True), (False, False)])
def test_shared_prefix(flint, oracle, N, H, Hk, L, S, D, P, lens, is_bf16, tokens):
    c = Cache(flint, oracle, 5 + L + S + P, N, H, Hk, L, S, D, is_bf16, lens, tokens, P=P)
    t = c.device()
    flint.attention_shared_prefix(t["q"], t["prefix_k"], t["prefix_v"], t["k"], t["v"], t["lens"], t["out"])
    got = c.read(t["out"])
    flint.synchronize()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), lens, prefix_k=c.value("prefix_k"), prefix_v=c.value("prefix_v"))
    check_out(got, want, size, score, S + P, is_bf16, "prefix")


WEIGHTS = [
    # N, H, Hk, L, S, D, lens
    (1, 1, 1, 1, 1, 64, None),
    (3, 6, 2, 1, 300, 128, [300, 0, 77]),
    (2, 40, 2, 1, 129, 64, None),                # two tiles of query heads
    (2, 4, 2, 6, 517, 64, [517, 3]),
    (1, 4, 4, 1, 6000, 128, [5999]),
    (2, 4, 1, 150, 150, 128, [150, 149]),
    (1, 6, 2, 333, 700, 64, [611]),
    (2, 2, 2, 700, 500, 128, [500, 130]),        # queries before every key
    (2, 12, 2, 7, 1001, 128, [1001, 600]),       # stored scores of three tiles of rows
    (1, 150, 1, 2, 130, 64, None),
    (1, 2, 1, 200, 5000, 64, [4990]),            # keys whose queries' blocks are few
]


@pytest.mark.parametrize("N,H,Hk,L,S,D,lens", WEIGHTS)
@pytest.mark.parametrize("is_bf16,tokens", [(True, True), (False, False)])
def test_weights(flint, oracle, N, H, Hk, L, S, D, lens, is_bf16, tokens):
    F = flint
    c = Cache(F, oracle, 3 + L + S + H, N, H, Hk, L, S, D, is_bf16, lens, tokens)
    t = c.device()
    before = np.random.default_rng(1).random((N, Hk, S)).astype(np.float32)
    room = dev(F, np.concatenate([before, np.full((N, Hk, 3), 7.0, np.float32)], axis=2), F.DType.FLOAT)
    w_in, w_out = dev(F, before, F.DType.FLOAT), room.view_as((N, Hk, S), (Hk * (S + 3), S + 3, 1))
    F.attention_weights(t["q"], t["k"], t["v"], w_in, t["lens"], w_out, t["out"])
    got, got_w = c.read(t["out"]), room.numpy()
    F.attention_weights(t["q"], t["k"], t["v"], w_in, t["lens"], out=t["out"])  # in place
    assert np.array_equal(w_in.numpy(), got_w[:, :, :S])
    F.synchronize()
    assert (got_w[:, :, S:] == 7.0).all()
    want, weights, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), lens)
    check_out(got, want, size, score, S, is_bf16, "weights' output")
    tol = (2 * (D + 4) * 2.0 ** -23 * score.max() + 2.0 ** -20 + 2.0 ** -13 + (S + H // Hk * L) * 2.0 ** -23) * weights + 2.0 ** -23 * (before + weights)
    off = np.abs(got_w[:, :, :S] - (before + weights)) / tol
    assert off.max() <= 1.0, f"{off.max():.2f} of the tolerance"


@pytest.mark.parametrize("L,S,window,sinks,length", [(1, 200, 50, 4, 150), (4, 200, 50, 4, 150), (160, 400, 60, 5, 390), (300, 300, 300, 0, 300)])
@pytest.mark.parametrize("is_bf16", [True, False])
def test_what_is_not_seen_may_be_anything(flint, oracle, L, S, window, sinks, length, is_bf16):
    """NaN and infinities past a sequence's length, before every window, and in keys that some queries see: they reach
    the queries that see them and no others."""
    H, Hk, D = 4, 2, 128
    c = Cache(flint, oracle, 77, 1, H, Hk, L, S, D, is_bf16, [length])
    nan, inf = (0x7FC0, 0x7F80) if is_bf16 else (0x7E00, 0x7C00)
    see = C.seen(L, length, window, sinks, S)
    for j in np.nonzero(~see.any(0))[0]:
        c.bits["k"][:, :, j] = nan if j % 2 else inf
        c.bits["v"][:, :, j] = nan if j % 3 else inf
    some = np.nonzero(see.any(0) & ~see.all(0))[0]
    if len(some) > 8:
        c.bits["v"][0, 0, some[len(some) // 2], 5] = nan
        c.bits["v"][0, 1, some[-2], 64] = inf
        c.bits["k"][0, 1, some[2], 3] = nan
    t = c.device()
    flint.attention_window(t["q"], t["k"], t["v"], window, sinks, t["lens"], t["out"])
    got = c.read(t["out"])
    flint.synchronize()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), [length], window, sinks)
    score, size = np.nan_to_num(score, posinf=0.0), np.where(np.isfinite(size), size, 0.0)
    check_out(got, want, size, score, S, is_bf16, "unseen")
    assert np.isfinite(got).any()


def test_values_that_some_see_beside_sequences_without_keys(flint, oracle):
    """More sequences than the GPU runs at a time, two of three without keys: a NaN that some queries of each of the
    others see reaches those queries, whichever sequences are worked on after one another."""
    N, L, S, D = 900, 40, 96, 64
    rng = np.random.default_rng(5)
    lens = np.where(rng.integers(0, 3, N) > 0, 0, rng.integers(60, S + 1, N))
    c = Cache(flint, oracle, 78, N, 1, 1, L, S, D, True, lens)
    for n in range(N):
        c.bits["v"][n, 0, max(lens[n] - 7, 0), n % D] = 0x7FC0
    t = c.device()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), lens, S, 0)
    size = np.where(np.isfinite(size), size, 0.0)
    for _ in range(3):
        flint.attention_window(t["q"], t["k"], t["v"], S, 0, t["lens"], t["out"])
        got = c.read(t["out"])
        flint.synchronize()
        check_out(got, want, size, score, S, True, "beside empty ones")


@pytest.mark.parametrize("L", [1, 200])
def test_peaked_scores_and_equal_results(flint, oracle, L):
    """Scores far apart, so that the running maximum moves; the same call twice gives the same bits."""
    c = Cache(flint, oracle, 8, 2, 4, 2, L, 1500, 128, True, [1500, 700], spread=4.0)
    t = c.device()
    flint.attention_window(t["q"], t["k"], t["v"], 900, 10, t["lens"], t["out"])
    got = c.read(t["out"])
    flint.attention_window(t["q"], t["k"], t["v"], 900, 10, t["lens"], t["out"])
    assert np.array_equal(got, c.read(t["out"]))
    flint.synchronize()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), [1500, 700], 900, 10)
    check_out(got, want, size, score, 1500, True, "peaked")


def test_a_length_outside_the_cache_counts_as_the_nearest(flint, oracle):
    c = Cache(flint, oracle, 9, 3, 2, 1, 2, 50, 64, True, [-5, 51, 2 ** 31 - 1])
    t = c.device()
    flint.attention_window(t["q"], t["k"], t["v"], 20, 1, t["lens"], t["out"])
    got = c.read(t["out"])
    flint.synchronize()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), [0, 50, 50], 20, 1)
    check_out(got, want, size, score, 21, True, "lengths")


@pytest.mark.parametrize("L", [1, 40])
def test_offsets_past_32_bits(flint, oracle, L):
    """Sequences of a cache that lie 3 GiB apart, the third past 2^31 elements from its start."""
    import torch
    F, O = flint, oracle
    H, Hk, S, D, apart = 4, 2, 300, 64, 3 << 29
    rng = np.random.default_rng(L)
    store = torch.empty(2 * apart + Hk * S * D, dtype=torch.bfloat16, device="cuda")
    q, k, v = (O.narrow(rng.standard_normal((3, h, n, D)).astype(np.float32), True) for h, n in ((H, L), (Hk, S), (Hk, S)))
    at = {}
    for name, a in (("k", k), ("v", v)):
        for n in range(3):
            store[n * apart:n * apart + Hk * S * D] = torch.from_numpy(a[n].reshape(-1).view(np.int16)).cuda().view(torch.bfloat16)
        t = F.Tensor.from_device_ptr(store.data_ptr(), (3, Hk, S, D), F.DType.BFLOAT16, keepalive=store, stride=(apart, S * D, D, 1), numel=store.numel())
        if name == "k":  # (v in storage of its own, as far apart)
            store = torch.empty_like(store)
        at[name] = t
    torch.cuda.synchronize()
    widen = lambda a: O.widen(a, True).astype(np.float64)  # noqa: E731
    out = F.attention_window(dev(F, q, F.DType.BFLOAT16), at["k"], at["v"], 200, 3)
    want, _, size, score = C.attention(widen(q), widen(k), widen(v), None, 200, 3)
    check_out(widen(out.numpy()), want, size, score, 203, True, "far apart")
    w, fresh = dev(F, rng.random((3, Hk, S)).astype(np.float32), F.DType.FLOAT), torch.empty(3, Hk, 100, D, dtype=torch.bfloat16, device="cuda")
    ko = F.Tensor.from_device_ptr(fresh.data_ptr(), (3, Hk, 100, D), F.DType.BFLOAT16, keepalive=fresh)
    F.cache_evict(at["k"], at["v"], w, 100, 10, k_out=ko)
    kept = C.evict(w.numpy(), None, 100, 10)
    F.synchronize()
    assert np.array_equal(ko.numpy()[2, 1], k[2, 1, kept[2, 1]])


def test_calls_from_two_threads(flint, oracle):
    """Calls of different shapes at once: the workspace is theirs in turn."""
    import threading
    F = flint
    cases = [Cache(F, oracle, 5, 2, 4, 2, 1, 3000, 128, True, [3000, 1111]), Cache(F, oracle, 6, 1, 6, 2, 150, 800, 64, False, [777])]
    devices, results = [c.device() for c in cases], [[], []]
    wants = [C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens) for c in cases]
    weights = [np.zeros((c.shape[0], c.shape[2], c.shape[4]), np.float32) for c in cases]

    def work(i):
        t = devices[i]
        for _ in range(20):
            w = dev(F, weights[i], F.DType.FLOAT)
            out, w = F.attention_weights(t["q"], t["k"], t["v"], w, t["lens"])
            results[i].append((out.numpy(), w.numpy()))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    F.synchronize()
    for i, c in enumerate(cases):
        want, _, size, score = wants[i]
        assert len(results[i]) == 20
        check_out(oracle.widen(results[i][0][0], c.is_bf16).astype(np.float64), want, size, score, c.shape[4], c.is_bf16, f"thread {i}")
        assert all(np.array_equal(a, results[i][0][0]) and np.array_equal(b, results[i][0][1]) for a, b in results[i])


EVICT = [
    # N, Hk, S, D, keep, recent, room, lens
    (1, 1, 1, 64, 1, 0, 1, None),
    (3, 2, 517, 64, 100, 17, 130, [517, 90, 101]),
    (2, 3, 3000, 128, 1025, 1025, 1025, [3000, 1026]),   # the recent ones alone
    (2, 1, 2500, 24, 1200, 0, 1300, [2500, 0]),          # none of them; a sequence without keys
    (1, 2, 100, 8, 100, 5, 100, None),                   # nothing to evict
    (2, 1, 60000, 8, 777, 20, 777, [60000, 30011]),      # more weights than fit in shared memory
    (1, 1, 30000, 8, 20000, 9000, 20000, None),          # ... or with a list beside them
    (2, 1, 22000, 8, 9000, 300, 9000, [22000, 16684]),   # more than a CTA holds in registers, listed, and as many as it does
    (1, 1, 16685, 8, 400, 300, 400, None),               # one more
]


@pytest.mark.parametrize("N,Hk,S,D,keep,recent,room,lens", EVICT)
@pytest.mark.parametrize("kind", ["spread", "equal", "odd"])
def test_evict(flint, oracle, N, Hk, S, D, keep, recent, room, lens, kind):
    """Bit for bit, with weights that are all different, mostly equal, or negative, infinite and NaN."""
    F = flint
    rng = np.random.default_rng(S + keep)
    k, v = (rng.integers(0, 2 ** 16, (N, Hk, S, D), dtype=np.uint16) for _ in range(2))
    w = rng.random((N, Hk, S)).astype(np.float32)
    if kind == "equal":
        w = np.floor(w * 4).astype(np.float32) / 4
    if kind == "odd":
        w = (w - 0.5) * 1e-38
        w[:, :, ::7] = np.nan
        w[:, :, 1::11] = np.inf
        w[:, :, 2::11] = -np.inf
        w[:, :, 3::5] = -0.0
        w[:, :, 4::5] = 0.0
    bf = F.DType.BFLOAT16
    store = dev(F, np.ascontiguousarray(k.transpose(0, 2, 1, 3)), bf)  # a token-major cache
    tk = store.view_as((N, Hk, S, D), (S * Hk * D, D, Hk * D, 1))
    tv, tw = dev(F, v, bf), dev(F, w, F.DType.FLOAT)
    ko, vo = dev(F, np.full((N, Hk, room, D), 0xABCD, np.uint16), bf), dev(F, np.full((N, Hk, room, D), 0x1234, np.uint16), bf)
    wo, kept = dev(F, np.full((N, Hk, room), 9.0, np.float32), F.DType.FLOAT), dev(F, np.full((N, Hk, keep), 5, np.int32), F.DType.INT32)
    tl = None if lens is None else dev(F, np.asarray(lens, np.int32), F.DType.INT32)
    F.cache_evict(tk, tv, tw, keep, recent, tl, ko, vo, wo, tl, kept)  # the new lengths in place of the old
    got = kept.numpy()
    F.synchronize()
    want = C.evict(w, lens, keep, recent)
    assert np.array_equal(got, want)
    if tl is not None:
        assert np.array_equal(tl.numpy(), np.minimum(lens, keep))
    gk, gv, gw = ko.numpy(), vo.numpy(), wo.numpy()
    for n in range(N):
        for h in range(Hk):
            at = want[n, h][want[n, h] >= 0]
            assert np.array_equal(gk[n, h, :len(at)], k[n, h, at]) and np.array_equal(gv[n, h, :len(at)], v[n, h, at])
            assert (gk[n, h, len(at):] == 0xABCD).all() and (gv[n, h, len(at):] == 0x1234).all()  # left as they were
            assert np.array_equal(gw[n, h, :len(at)].view(np.uint32), w[n, h, at].view(np.uint32))
            assert (gw[n, h, len(at):] == 0).all()
    ko2, _, _, _ = F.cache_evict(tk, tv, tw, keep, recent)  # outputs made by the wrapper, positions not wanted
    full = C.evict(w, None, keep, recent)
    assert np.array_equal(ko2.numpy()[0, 0, :min(keep, S)], k[0, 0, full[0, 0][full[0, 0] >= 0]])
    F.synchronize()


def test_a_decoder_that_evicts(flint, oracle):
    """A prompt behind a shared prefix, then tokens one by one: attention that keeps the books, eviction when the
    cache is full, and on with what is left, as a program would use them together."""
    F = flint
    rng = np.random.default_rng(31)
    N, H, Hk, D, S, L0, keep, recent = 2, 4, 2, 64, 48, 40, 24, 8
    bf = F.DType.BFLOAT16
    narrow = lambda *shape: oracle.narrow(rng.standard_normal(shape).astype(np.float32), True)  # noqa: E731
    widen = lambda a: oracle.widen(a, True).astype(np.float64)  # noqa: E731
    k, v = np.zeros((N, Hk, S, D), np.uint16), np.zeros((N, Hk, S, D), np.uint16)
    k[:, :, :L0], v[:, :, :L0] = narrow(N, Hk, L0, D), narrow(N, Hk, L0, D)
    tk, tv, lens = dev(F, k, bf), dev(F, v, bf), np.full(N, L0, np.int32)
    spare_k, spare_v, weights = F.Tensor.empty((N, Hk, S, D), bf), F.Tensor.empty((N, Hk, S, D), bf), dev(F, np.zeros((N, Hk, S), np.float32), F.DType.FLOAT)
    spare_w = F.Tensor.empty((N, Hk, S), F.DType.FLOAT)
    pk, pv = narrow(1, Hk, 70, D), narrow(1, Hk, 70, D)
    book = np.zeros((N, Hk, S))

    q = narrow(N, H, L0, D)
    got = F.attention_shared_prefix(dev(F, q, bf), dev(F, pk, bf), dev(F, pv, bf), tk, tv, dev(F, lens, F.DType.INT32)).numpy()
    want, _, size, score = C.attention(widen(q), widen(k), widen(v), lens, prefix_k=widen(pk), prefix_v=widen(pv))
    check_out(widen(got), want, size, score, S + 70, True, "prompt")
    evictions = 0
    for step in range(30):
        if lens[0] == S:
            tl = dev(F, lens, F.DType.INT32)
            host = weights.numpy()
            F.cache_evict(tk, tv, weights, keep, recent, tl, spare_k, spare_v, spare_w, tl)
            kept = C.evict(host, lens, keep, recent)
            for n in range(N):
                for h in range(Hk):
                    k[n, h, :keep], v[n, h, :keep] = k[n, h, kept[n, h]], v[n, h, kept[n, h]]
                    book[n, h, :keep], book[n, h, keep:] = book[n, h, kept[n, h]], 0
            (tk, spare_k), (tv, spare_v), (weights, spare_w) = (spare_k, tk), (spare_v, tv), (spare_w, weights)
            lens = tl.numpy()
            assert (lens == keep).all()
            evictions += 1
        at = int(lens[0])
        new_k, new_v = narrow(N, Hk, 1, D), narrow(N, Hk, 1, D)
        for cache, host, new in ((tk, k, new_k), (tv, v, new_v)):
            F.copy(dev(F, new, bf), cache.view_as((N, Hk, 1, D), (Hk * S * D, S * D, D, 1), at * D))
            host[:, :, at:at + 1] = new
        lens = lens + 1
        q = narrow(N, H, 1, D)
        tl = dev(F, lens, F.DType.INT32)
        out, _ = F.attention_weights(dev(F, q, bf), tk, tv, weights, tl)
        want, w, size, score = C.attention(widen(q), widen(k), widen(v), lens)
        book += w
        check_out(widen(out.numpy()), want, size, score, S, True, f"step {step}")
        near = F.attention_window(dev(F, q, bf), tk, tv, 12, 4, tl)
        want, _, size, score = C.attention(widen(q), widen(k), widen(v), lens, 12, 4)
        check_out(widen(near.numpy()), want, size, score, 16, True, f"window of step {step}")
    F.synchronize()
    assert evictions == 1 and np.abs(weights.numpy()[:, :, :int(lens[0])] - book[:, :, :int(lens[0])]).max() < 1e-4  # 30 steps of float sums near 1


SHORT_WALKS = [
    # N, H, Hk, L, S, D, window, lens: units of one step of 64 keys, several to a CTA
    (130, 8, 8, 1, 60, 64, 60, None),
    (130, 8, 8, 1, 700, 128, 64, [700 - 5 * n for n in range(130)]),
    (16, 8, 8, 1, 300, 128, 300, [300] + [40] * 15),
    (200, 6, 3, 2, 64, 64, 64, [n * 37 % 65 for n in range(200)]),
    (250, 35, 1, 1, 64, 64, 64, None),                               # three tiles of 16 rows, the last one partial
    (200, 70, 2, 1, 40, 128, 40, [n * 13 % 41 for n in range(200)]),
]


@pytest.mark.parametrize("N,H,Hk,L,S,D,window,lens", SHORT_WALKS)
def test_many_short_walks_one_after_the_other(flint, oracle, N, H, Hk, L, S, D, window, lens):
    """A CTA of the few-row kernel goes through many units, whose queries take turns in two places: right, and the same
    bits every time. (With the keys' weights the kernel takes up to 63 rows, in tiles of 16.)"""
    F = flint
    c = Cache(F, oracle, 21 + N + S, N, H, Hk, L, S, D, True, lens)
    t = c.device()
    weighed = window == S
    zeros = np.zeros((N, Hk, S), np.float32)

    def once():
        if not weighed:
            F.attention_window(t["q"], t["k"], t["v"], window, 0, t["lens"], t["out"])
            return c.read(t["out"]), zeros
        _, w = F.attention_weights(t["q"], t["k"], t["v"], dev(F, zeros, F.DType.FLOAT), t["lens"], out=t["out"])
        return c.read(t["out"]), w.numpy()

    got, got_w = once()
    for _ in range(20):
        again, again_w = once()
        assert np.array_equal(got, again) and np.array_equal(got_w, again_w)
    F.synchronize()
    want, weights, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), lens, window, 0)
    check_out(got, want, size, score, S, True, "short walks")
    if weighed:
        tol = (2 * (D + 4) * 2.0 ** -23 * score.max() + 2.0 ** -20 + 2.0 ** -13 + (S + H // Hk * L) * 2.0 ** -23) * weights
        assert (np.abs(got_w - weights) <= tol).all()


def put(c, name, at, value):
    """A value (nan, inf or -inf) at a place of an operand."""
    bits = {"nan": (0x7FC0, 0x7E00), "inf": (0x7F80, 0x7C00), "-inf": (0xFF80, 0xFC00)}[value]
    c.bits[name][at] = bits[0] if c.is_bf16 else bits[1]


@pytest.mark.parametrize("H,Hk,L,S", [(1, 1, 1, 1), (4, 2, 1, 100), (4, 2, 1, 3000), (6, 2, 4, 500), (4, 2, 40, 300)])
@pytest.mark.parametrize("route", ["window", "prefix", "weights"])
@pytest.mark.parametrize("is_bf16", [True, False])
def test_seen_infinities_reach_the_result(flint, oracle, H, Hk, L, S, route, is_bf16):
    """An infinity in a value that a query sees is its result's, whichever others see it too; both signs, or a NaN,
    make a NaN. Scores are close, so that no weight rounds to zero."""
    F, N, D, P = flint, 2, 64, 70
    c = Cache(F, oracle, 91 + S + L, N, H, Hk, L, S, D, is_bf16, [S, max(S // 2, 1)], P=P if route == "prefix" else 0, spread=0.5)
    last = S // 2 - 1 if S > 1 else 0  # seen by every query of the first sequence, by the last ones of the second
    put(c, "v", (0, 0, 0, 3), "inf")
    put(c, "v", (0, 0, S // 2, 4), "-inf")
    put(c, "v", (0, Hk - 1, S // 3, 5), "inf")
    put(c, "v", (0, Hk - 1, S // 2, 5), "-inf" if S > 1 else "inf")
    put(c, "v", (0, 0, S // 4, 6), "nan")
    put(c, "v", (1, 0, last, 7), "inf")
    put(c, "v", (1, Hk - 1, last // 2, 63), "-inf")
    if route == "prefix":
        put(c, "prefix_v", (0, 0, 0, 8), "inf")
        put(c, "prefix_v", (0, Hk - 1, P - 1, 9), "-inf")
        put(c, "prefix_v", (0, 0, 64, 3), "-inf")
    t = c.device()
    if route == "window":
        F.attention_window(t["q"], t["k"], t["v"], S, 0, t["lens"], t["out"])
        got = c.read(t["out"])
        F.attention_window(t["q"], t["k"], t["v"], max(S // 2, 1), 1, t["lens"], t["out"])
        under = c.read(t["out"])
        with np.errstate(invalid="ignore"):
            want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens, max(S // 2, 1), 1)
        check_out(under, want, np.nan_to_num(size, posinf=0.0), score, S, is_bf16, "under a window")
        with np.errstate(invalid="ignore"):
            want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens)
    elif route == "prefix":
        F.attention_shared_prefix(t["q"], t["prefix_k"], t["prefix_v"], t["k"], t["v"], t["lens"], t["out"])
        got = c.read(t["out"])
        with np.errstate(invalid="ignore"):
            want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens, prefix_k=c.value("prefix_k"), prefix_v=c.value("prefix_v"))
    else:
        w = dev(F, np.zeros((N, Hk, S), np.float32), F.DType.FLOAT)
        F.attention_weights(t["q"], t["k"], t["v"], w, t["lens"], out=t["out"])
        got = c.read(t["out"])
        with np.errstate(invalid="ignore"):
            want, weights, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens)
        tol = (2 * (D + 4) * 2.0 ** -23 * score.max() + 2.0 ** -20 + 2.0 ** -13 + (S + H // Hk * L) * 2.0 ** -23) * weights
        assert (np.abs(w.numpy() - weights) <= tol).all()  # values have no part in them
    F.synchronize()
    check_out(got, want, np.nan_to_num(size, posinf=0.0), score, S + P, is_bf16, route)
    assert np.isinf(got).any()


@pytest.mark.parametrize("L,S,window,sinks,lens", [(1, 300, 100, 5, [300, 250]), (5, 300, 100, 5, [300, 103]), (40, 300, 300, 0, [300, 170]),
                                                   (150, 500, 200, 20, [500, 490]), (60, 9000, 9000, 0, [9000, 4000])])
def test_large_values_of_unseen_keys(flint, oracle, L, S, window, sinks, lens):
    """Finite values far above the others in keys that some queries see and others do not: those others' results have
    nothing of them. (2^-126, the least normal float, times 1e37 would be 0.1.)"""
    c = Cache(flint, oracle, 55 + L, 2, 4, 2, L, S, 64, True, lens, spread=0.5)
    large = oracle.narrow(np.array([1e37], np.float32), True)[0]
    for n, length in enumerate(lens):
        at = max(length - max(L // 2, 1) - 4, 0)
        c.bits["v"][n, 0, at:at + 8, 7] = large           # the later queries see them
        before = length - window - L // 2
        if before > sinks + 8:
            c.bits["v"][n, 1, before - 4:before + 4, 9] = large  # the earlier ones
        c.bits["v"][n, 1, sinks:sinks + 8, 11] = large    # not in the sinks
    t = c.device()
    flint.attention_window(t["q"], t["k"], t["v"], window, sinks, t["lens"], t["out"])
    got = c.read(t["out"])
    flint.synchronize()
    want, _, size, score = C.attention(c.value("q"), c.value("k"), c.value("v"), lens, window, sinks)
    check_out(got, want, size, score, S, True, "large values")
    small = np.abs(want).max(-1) < 100
    assert np.linalg.norm(got[small] - want[small]) <= 5e-3 * np.linalg.norm(want[small])


@pytest.mark.parametrize("H,Hk,L,S,D", [(6, 2, 1, 300, 64), (6, 2, 150, 400, 64), (4, 1, 33, 300, 128), (14, 2, 100, 350, 128), (8, 2, 200, 600, 64)])
@pytest.mark.parametrize("is_bf16", [True, False])
def test_weights_of_keys_that_every_query_scores_minus_infinity(flint, oracle, H, Hk, L, S, D, is_bf16):
    """Such keys weigh nothing, with blocks of rows that are full and that are not (groups of 3 and 7; a last block's end)."""
    F = flint
    c = Cache(F, oracle, 71 + L, 2, H, Hk, L, S, D, is_bf16, [S, S - 30], spread=0.5)
    c.bits["q"][..., 9] &= 0x7FFF  # positive
    _, _, _, score = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens)
    tiny = c.bits["q"][..., 9] == 0
    c.bits["q"][..., 9][tiny] = 0x3C00
    at = [0, 100, S - 31 - L // 2, S - 1 - L // 2]
    for n in range(2):
        for h in range(Hk):
            for j in at:
                put(c, "k", (n, h, j, 9), "-inf")
    t = c.device()
    w = dev(F, np.zeros((2, Hk, S), np.float32), F.DType.FLOAT)
    F.attention_weights(t["q"], t["k"], t["v"], w, t["lens"], out=t["out"])
    got, got_w = c.read(t["out"]), w.numpy()
    F.synchronize()
    want, weights, size, _ = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens)
    assert (got_w[:, :, at] == 0).all()
    tol = (2 * (D + 4) * 2.0 ** -23 * score.max() + 2.0 ** -20 + 2.0 ** -13 + (S + H // Hk * L) * 2.0 ** -23) * weights
    assert (np.abs(got_w - weights) <= tol).all()
    check_out(got, want, size, score, S, is_bf16, "beside them")


@pytest.mark.parametrize("H,Hk,L,S,D", [(6, 2, 1, 300, 64), (6, 2, 150, 400, 64), (8, 2, 200, 600, 64)])
@pytest.mark.parametrize("odd", ["nan", "inf"])
def test_weights_beside_scores_without_a_softmax(flint, oracle, H, Hk, L, S, D, odd):
    """A key that some queries score NaN or +inf takes these queries' weights with it, and no others: those of every key
    they see, one that everything scores -inf among them."""
    F = flint
    c = Cache(F, oracle, 72 + L, 2, H, Hk, L, S, D, True, [S, S - 30], spread=0.5)
    c.bits["q"][..., 9] = c.bits["q"][..., 9] & 0x7FFF | 0x3800  # positive
    put(c, "k", (0, 0, S - 1 - L // 2, 9), odd)
    for h in range(Hk):
        put(c, "k", (0, h, 50, 9), "-inf")
    t = c.device()
    w = dev(F, np.zeros((2, Hk, S), np.float32), F.DType.FLOAT)
    F.attention_weights(t["q"], t["k"], t["v"], w, t["lens"], out=t["out"])
    got, got_w = c.read(t["out"]), w.numpy()
    F.synchronize()
    with np.errstate(invalid="ignore"):
        want, weights, _, _ = C.attention(c.value("q"), c.value("k"), c.value("v"), c.lens)
    assert np.array_equal(np.isnan(got_w), np.isnan(weights)) and np.isnan(weights[0, 0]).all() and not np.isnan(weights[0, 1:]).any()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and (got_w[0, 1:, 50] == 0).all()


@pytest.mark.parametrize("S,P", [(65536, 0), (700, 65536)])
@pytest.mark.parametrize("is_bf16", [True, False])
def test_many_light_keys_beside_a_heavy_one(flint, oracle, S, P, is_bf16):
    """One key takes nearly all of the weight, and each of the others about 2^-26, below what a half holds, in a walk that
    is not divided: together they are seen in the columns where the heavy key's value is zero. A half weight is off by
    2^-32 at most of the largest, times values below 1."""
    F, H, L, D = flint, 64, 600, 64
    c = Cache(F, oracle, 61, 1, H, 1, L, S, D, is_bf16, None, P=P, spread=0.1)
    keys, values = ("prefix_k", "prefix_v") if P else ("k", "v")
    c.bits["q"][..., 0] = oracle.narrow(np.array([16.0], np.float32), is_bf16)[0]
    for name in {keys, "k"}:
        c.bits[name][..., 0] = 0
    c.bits[keys][0, 0, 5, 0] = oracle.narrow(np.array([9.0], np.float32), is_bf16)[0]
    for name in {values, "v"}:
        c.bits[name] = oracle.narrow(np.abs(np.random.default_rng(2).standard_normal(c.bits[name].shape)).clip(0, 1).astype(np.float32), is_bf16)
    c.bits[values][0, 0, 5] = 0
    t = c.device()
    if P:
        F.attention_shared_prefix(t["q"], t["prefix_k"], t["prefix_v"], t["k"], t["v"], None, t["out"])
    else:
        F.attention_window(t["q"], t["k"], t["v"], S, 0, None, t["out"])
    got = c.read(t["out"])
    F.synchronize()
    u = 2.0 ** (-8 if is_bf16 else -11)
    q, k, v = c.value("q")[0], c.value("k")[0, 0], c.value("v")[0, 0]
    for h, i in ((0, 0), (3, 77), (63, 599), (20, 300)):
        seen_k, seen_v = k[:i + S - L + 1], v[:i + S - L + 1]
        if P:
            seen_k, seen_v = np.concatenate([c.value("prefix_k")[0, 0], seen_k]), np.concatenate([c.value("prefix_v")[0, 0], seen_v])
        want, _, size, score = C.attend(q[h, i], seen_k, seen_v)
        n = len(seen_k)
        tol = u * want + (u + 2 * (D + 4) * 2.0 ** -23 * score + 2.0 ** -12 + n * 2.0 ** -23) * size + (0.0 if is_bf16 else n * 2.0 ** -32 + 2.0 ** -25)
        assert (want > 4e-4).all() and (np.abs(got[0, h, i] - want) <= tol).all(), (np.abs(got[0, h, i] - want) / tol).max()


@pytest.mark.parametrize("N,H,Hk,L,S,D,P,lens", [
    (5, 17, 1, 1, 40, 64, 300, [40, 0, 7, 33, 12]),
    (6, 8, 2, 5, 70, 128, 700, [70, 4, 5, 0, 61, 33]),
    (4, 16, 2, 5, 90, 64, 515, [90, 90, 3, 64]),
    (3, 127, 1, 1, 50, 128, 260, [50, 1, 0]),
    (3, 8, 2, 16, 64, 64, 1000, [64, 15, 16]),
])
@pytest.mark.parametrize("is_bf16,tokens", [(True, True), (False, False)])
def test_a_few_tokens_of_several_sequences_behind_a_prefix(flint, oracle, N, H, Hk, L, S, D, P, lens, is_bf16, tokens):
    """17 to 127 rows to a key-value head: a speculated step, or many query heads to one of keys."""
    test_shared_prefix(flint, oracle, N, H, Hk, L, S, D, P, lens, is_bf16, tokens)


def test_eviction_into_a_cache_with_keys_beside_values(flint, oracle):
    """(N, room, 2, kv_heads, D): the outputs take turns in memory, and rows past the new length stay as they were."""
    F, N, Hk, S, D, keep, recent, room = flint, 2, 3, 700, 64, 333, 30, 400
    rng = np.random.default_rng(8)
    k, v = (rng.integers(0, 2 ** 16, (N, Hk, S, D), dtype=np.uint16) for _ in range(2))
    w, lens, bf = rng.random((N, Hk, S)).astype(np.float32), [700, 250], F.DType.BFLOAT16
    store = dev(F, np.full((N, room, 2, Hk, D), 0xABCD, np.uint16), bf)
    ko, vo = (store.view_as((N, Hk, room, D), (room * 2 * Hk * D, D, 2 * Hk * D, 1), i * Hk * D) for i in range(2))
    kept = dev(F, np.zeros((N, Hk, keep), np.int32), F.DType.INT32)
    _, _, wo, lo = F.cache_evict(dev(F, k, bf), dev(F, v, bf), dev(F, w, F.DType.FLOAT), keep, recent, dev(F, np.asarray(lens, np.int32), F.DType.INT32), ko, vo, kept=kept)
    got, want = store.numpy(), C.evict(w, lens, keep, recent)
    F.synchronize()
    assert np.array_equal(kept.numpy(), want) and np.array_equal(lo.numpy(), [333, 250])
    for n in range(N):
        for h in range(Hk):
            at = want[n, h][want[n, h] >= 0]
            for i, source in enumerate((k, v)):
                assert np.array_equal(got[n, :len(at), i, h], source[n, h, at]) and (got[n, len(at):, i, h] == 0xABCD).all()
            assert np.array_equal(wo.numpy()[n, h, :len(at)], w[n, h, at])
