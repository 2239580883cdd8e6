"""Cases for the operators on a decoder's key-value cache: attention with a sliding window and sinks, attention of a batch
that shares a prefix, attention that adds up the keys' weights, and eviction by those weights.

`run` computes a case in plain torch operations in 32 bits, or, where `own` is set, with the library's kernels."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # A short chat turn's single token: latency alone.
        dict(name="window_one_token", op="window", type="fp16", N=1, H=8, KVH=2, D=64, L=1, S=77, W=64, sinks=4, ragged=False, layout="heads"),
        # A serving batch's decode step under a window of half the cache.
        dict(name="window_decode_batch", op="window", type="bf16", N=32, H=32, KVH=8, D=128, L=1, S=8192, W=4096, sinks=4, ragged=True, layout="heads"),
        # One token of one very long sequence that sees all of it: the keys are split over the whole GPU.
        dict(name="window_decode_long", op="window", type="bf16", N=1, H=32, KVH=8, D=128, L=1, S=131072, W=131072, sinks=0, ragged=False, layout="tokens"),
        # A long prompt's prefill under a window.
        dict(name="window_prefill_long", op="window", type="bf16", N=1, H=32, KVH=8, D=128, L=8192, S=8192, W=1024, sinks=16, ragged=False, layout="tokens"),
        # A padded batch of prompt chunks of odd sizes; the shortest sequences leave queries without keys.
        dict(name="window_chunks_ragged", op="window", type="fp16", N=5, H=12, KVH=4, D=64, L=333, S=1511, W=300, sinks=7, ragged=True, layout="heads"),
        # A batch of samples of one prompt, a few tokens each.
        dict(name="prefix_few_samples", op="prefix", type="fp16", N=3, H=8, KVH=1, D=64, L=1, P=257, S=40, ragged=True, layout="heads"),
        # A decode step of many conversations behind one long system prompt.
        dict(name="prefix_decode_batch", op="prefix", type="bf16", N=64, H=32, KVH=8, D=128, L=1, P=8192, S=512, ragged=True, layout="heads"),
        # Questions of some hundred tokens, each appended to the same document.
        dict(name="prefix_extend", op="prefix", type="bf16", N=8, H=16, KVH=16, D=128, L=250, P=4096, S=300, ragged=True, layout="tokens"),
        # A decode step that keeps the books for eviction.
        dict(name="weights_decode_batch", op="weights", type="bf16", N=16, H=32, KVH=8, D=128, L=1, S=4096, ragged=True, layout="heads"),
        # A prompt's prefill that keeps them.
        dict(name="weights_prefill", op="weights", type="fp16", N=2, H=16, KVH=4, D=64, L=2048, S=2048, ragged=False, layout="tokens"),
        # A cache of odd sizes cut down.
        dict(name="evict_small", op="evict", type="fp16", N=3, KVH=2, D=64, S=517, keep=100, recent=17, ragged=True, layout="heads"),
        # A serving batch's caches halved.
        dict(name="evict_batch", op="evict", type="bf16", N=16, KVH=8, D=128, S=8192, keep=4096, recent=256, ragged=True, layout="heads"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "prefix", "weights", "evict"])
    D = rng.choice([64, 128])
    KVH = rng.choice([1, 2, 3, 4, 8])
    G = rng.choice([1, 2, 3, 4, 7, 8])
    case = dict(op=op, type=rng.choice(["bf16", "fp16"]), D=D, KVH=KVH, ragged=rng.random() < 0.7, layout=rng.choice(["heads", "tokens"]))
    if op == "evict":
        N, S = _log(rng, 1, 32), _log(rng, 16, 16384)
        N = max(1, min(N, (16 * 8 * 8192 * 128) // (KVH * S * D)))
        keep = rng.randint(1, S)
        return dict(case, N=N, S=S, keep=keep, recent=rng.randint(0, keep))
    H = KVH * G
    if rng.random() < 0.5:  # single tokens, or the few of a speculated step
        L = rng.choice([1, 1, 1, 2, 5])
        N, S = _log(rng, 1, 64), _log(rng, 16, 32768)
        N = max(1, min(N, (64 << 20) // (KVH * S * D)))
    else:
        N, S = _log(rng, 1, 8), _log(rng, 64, 4096)
        L = rng.randint(1, S)
        while N > 1 and N * H * L * S > (1 << 28):
            N -= 1
    case.update(N=N, H=H, L=L, S=S)
    if op == "window":
        case.update(W=_log(rng, 1, 2 * S), sinks=rng.choice([0, 1, 4, 16, 130]))
    if op == "prefix":
        case.update(P=_log(rng, 16, 8192))
        while case["N"] > 1 and case["N"] * H * L * (case["P"] + S) > (1 << 28):
            case["N"] -= 1
    return case


def lengths(case):
    """The sequences' lengths: all S, or spread between an eighth of S and S in no order, the first as long as the cache."""
    N, S = case["N"], case["S"]
    if not case["ragged"]:
        return [S] * N
    return [S - (n * 5 % N) * (S - S // 8) // max(N, 1) for n in range(N)]


def _stored(case, gen, dtype, N, heads, length, D):
    """A (N, heads, length, D) view of random values, head-major or token-major in memory."""
    if case["layout"] == "tokens":
        return torch.randn(N, length, heads, D, device="cuda", generator=gen, dtype=dtype).transpose(1, 2)
    return torch.randn(N, heads, length, D, device="cuda", generator=gen, dtype=dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, N, KVH, S, D = TYPES[case["type"]], case["N"], case["KVH"], case["S"], case["D"]
    state = dict(case=case)
    t = state["t"] = {}
    t["lens"] = torch.tensor(lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    t["k"] = _stored(case, gen, dtype, N, KVH, S, D)
    t["v"] = _stored(case, gen, dtype, N, KVH, S, D)
    if case["op"] == "evict":
        # Weights added up over many steps: a few heavy keys among many light ones, some of them equal.
        w = torch.rand(N, KVH, S, device="cuda", generator=gen).pow(8) * 20
        t["weights"] = (w * 64).round() / 64
        keep = case["keep"]
        t["k_out"], t["v_out"] = (torch.zeros(N, KVH, keep, D, dtype=dtype, device="cuda") for _ in range(2))
        t["weights_out"] = torch.zeros(N, KVH, keep, device="cuda")
        t["lens_out"] = torch.zeros(N, dtype=torch.int32, device="cuda")
        t["kept"] = torch.zeros(N, KVH, keep, dtype=torch.int32, device="cuda")
    else:
        L, H = case["L"], case["H"]
        t["q"] = _stored(case, gen, dtype, N, H, L, D)
        t["out"] = torch.zeros_like(t["q"])
        if case["op"] == "prefix":
            t["prefix_k"] = _stored(case, gen, dtype, 1, KVH, case["P"], D)
            t["prefix_v"] = _stored(case, gen, dtype, 1, KVH, case["P"], D)
        if case["op"] == "weights":
            t["weights"] = torch.rand(N, KVH, S, device="cuda", generator=gen) * 3
            t["weights_out"] = torch.zeros(N, KVH, S, device="cuda")
    if own:  # the views of its buffers that a program makes once
        state["f"] = {name: _wrap(x) for name, x in t.items() if x is not None}
    return state


def _wrap(x):
    from libwaifu_b200 import flint as F
    types = {torch.bfloat16: F.DType.BFLOAT16, torch.float16: F.DType.FLOAT16, torch.float32: F.DType.FLOAT, torch.int32: F.DType.INT32}
    return F.Tensor.from_device_ptr(x.data_ptr(), tuple(x.shape), types[x.dtype], keepalive=x, stride=tuple(x.stride()), numel=x.numel())


def run(state):
    case, t = state["case"], state["t"]
    if own:
        return _run_own(case, t, state["f"])
    if case["op"] == "evict":
        return _evict(case, t)
    q, k, v = t["q"].float(), t["k"].float(), t["v"].float()
    N, H, L, D = q.shape
    KVH, S = k.shape[1], k.shape[2]
    G = H // KVH
    lens = t["lens"].long() if t["lens"] is not None else torch.full((N,), S, device="cuda")
    j = torch.arange(S, device="cuda")
    p = torch.arange(L, device="cuda")[None, :] + lens[:, None] - L
    visible = (j <= p[:, :, None]) & (j < lens[:, None, None])
    if case["op"] == "window":
        visible &= (j > p[:, :, None] - case["W"]) | (j < case["sinks"])
    # Rows (group, query) of one key-value head in one product.
    q = (q * (1.0 / math.sqrt(D))).reshape(N, KVH, G * L, D)
    s = torch.matmul(q, k.transpose(2, 3)).reshape(N, KVH, G, L, S)
    s = s.masked_fill_(~visible[:, None, None], -math.inf)
    if case["op"] == "prefix":
        P = case["P"]
        pk, pv = t["prefix_k"].float()[0], t["prefix_v"].float()[0]
        rows = q.transpose(0, 1).reshape(KVH, N * G * L, D)
        shared = torch.matmul(rows, pk.transpose(1, 2)).reshape(KVH, N, G, L, P).transpose(0, 1)
        m = torch.maximum(shared.amax(-1, keepdim=True), s.amax(-1, keepdim=True))
        shared, s = (shared - m).exp(), (s - m).exp()
        total = shared.sum(-1, keepdim=True) + s.sum(-1, keepdim=True)
        o = torch.matmul(shared.transpose(0, 1).reshape(KVH, N * G * L, P), pv).reshape(KVH, N, G, L, D).transpose(0, 1)
        o = (o + torch.matmul(s.reshape(N, KVH, G * L, S), v).reshape(N, KVH, G, L, D)) / total
        return {"out": o.reshape(N, H, L, D).to(t["out"].dtype)}
    m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    s = s.sub_(m).exp_()
    w = s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-30))
    o = torch.matmul(w.reshape(N, KVH, G * L, S), v).reshape(N, H, L, D).to(t["out"].dtype)
    if case["op"] == "weights":
        return {"out": o, "weights": t["weights"] + w.sum((2, 3))}
    return {"out": o}


def _evict(case, t):
    keep, recent = case["keep"], case["recent"]
    k, v, w = t["k"], t["v"], t["weights"]
    N, KVH, S, D = k.shape
    lens = t["lens"].long() if t["lens"] is not None else torch.full((N,), S, device="cuda")
    j = torch.arange(S, device="cuda")
    rank = w.masked_fill((j >= lens[:, None] - recent)[:, None], math.inf).masked_fill((j >= lens[:, None])[:, None], -math.inf)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.where(torch.arange(keep, device="cuda") < lens[:, None, None], first, S).sort(-1).values
    there = kept < S
    at = torch.where(there, kept, 0)
    rows = at[..., None].expand(N, KVH, keep, D)
    return {"k": torch.gather(k, 2, rows) * there[..., None], "v": torch.gather(v, 2, rows) * there[..., None],
            "weights": torch.gather(w, 2, at) * there, "lens": lens.clamp(max=keep).int(), "kept": torch.where(there, kept, -1).int()}


def _run_own(case, t, f):
    from libwaifu_b200 import flint as F
    lens = f.get("lens")
    if case["op"] == "evict":
        F.cache_evict(f["k"], f["v"], f["weights"], case["keep"], case["recent"], lens, f["k_out"], f["v_out"], f["weights_out"], f["lens_out"], f["kept"])
        return {"k": t["k_out"], "v": t["v_out"], "weights": t["weights_out"], "lens": t["lens_out"], "kept": t["kept"]}
    if case["op"] == "window":
        F.attention_window(f["q"], f["k"], f["v"], case["W"], case["sinks"], lens, f["out"])
    elif case["op"] == "prefix":
        F.attention_shared_prefix(f["q"], f["prefix_k"], f["prefix_v"], f["k"], f["v"], lens, f["out"])
    else:
        F.attention_weights(f["q"], f["k"], f["v"], f["weights"], lens, f["weights_out"], f["out"])
        return {"out": t["out"], "weights": t["weights_out"]}
    return {"out": t["out"]}


def work(case):
    """Every key that some query sees read once, queries and results once; four operations per query head, visible key and
    position of head_dim (six where a long walk has to meet its scores twice)."""
    N, KVH, S, D = case["N"], case["KVH"], case["S"], case["D"]
    lens = lengths(case)
    if case["op"] == "evict":
        keep = case["keep"]
        rows = sum(min(n, keep) for n in lens) * KVH
        return {"bytes": 4 * KVH * sum(lens) + rows * (2 * 4 * D + 8) + 4 * N * KVH * keep, "flops": 0}
    H, L = case["H"], case["L"]
    W, sinks = (case["W"], case["sinks"]) if case["op"] == "window" else (S, 0)
    keys = pairs = 0
    for n in lens:
        first, last = max(n - L, 0), n - 1
        if n == 0:
            continue
        begin = max(first - W + 1, 0)  # of the first query's window; the windows from there on hold every key up to the last
        keys += n - begin + min(sinks, begin)
        p = torch.arange(first, n, dtype=torch.float64)
        low = (p - W + 1).clamp(min=0)
        pairs += float((p - low + 1 + torch.clamp(low, max=sinks)).sum())
    size = 2 * (2 * N * H * L * D) + 2 * (2 * KVH * keys * D)
    flops = 4 * H * pairs * D
    if case["op"] == "prefix":
        size += 2 * (2 * KVH * case["P"] * D)
        flops += 4.0 * N * H * L * case["P"] * D
    if case["op"] == "weights":
        size += 8 * N * KVH * S
    return {"bytes": size, "flops": flops}


def exact(case, seed):
    t = prepare(case, seed)["t"]
    N, KVH, S, D = case["N"], case["KVH"], case["S"], case["D"]
    lens = lengths(case)
    if case["op"] == "evict":
        keep, recent = case["keep"], case["recent"]
        weights = t["weights"].double().cpu().numpy()
        got = {"k": torch.zeros(N, KVH, keep, D, dtype=torch.float64), "v": torch.zeros(N, KVH, keep, D, dtype=torch.float64),
               "weights": torch.zeros(N, KVH, keep, dtype=torch.float64), "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32),
               "kept": torch.full((N, KVH, keep), -1, dtype=torch.int32)}
        for n in range(N):
            for h in range(KVH):
                row = weights[n, h]
                old = max(lens[n] - recent, 0)
                chosen = list(range(lens[n]))
                if lens[n] > keep:
                    by_weight = sorted(range(old), key=lambda i: (-row[i], i))
                    chosen = sorted(by_weight[:keep - recent] + list(range(old, lens[n])))
                at = torch.tensor(chosen, dtype=torch.long)
                got["kept"][n, h, :len(chosen)] = at.int()
                for name in ("k", "v", "weights"):
                    got[name][n, h, :len(chosen)] = t[name][n, h].index_select(0, at.cuda()).double().cpu()
        return got
    H, L, G = case["H"], case["L"], case["H"] // KVH
    out = torch.zeros(N, H, L, D, dtype=torch.float64)
    weights = t["weights"].double().cpu() if case["op"] == "weights" else None
    for n in range(N):
        for h in range(KVH):
            keys, values = t["k"][n, h, :lens[n]].double(), t["v"][n, h, :lens[n]].double()
            for g in range(G):
                scores = t["q"][n, h * G + g].double() @ keys.T / math.sqrt(D)
                ahead = torch.arange(lens[n], device="cuda")[None, :] - (torch.arange(L, device="cuda")[:, None] + lens[n] - L)
                hidden = ahead > 0
                if case["op"] == "window":
                    hidden |= (ahead <= -case["W"]) & (torch.arange(lens[n], device="cuda") >= case["sinks"])[None, :]
                scores[hidden] = -math.inf
                all_values = values
                if case["op"] == "prefix":
                    scores = torch.cat([t["q"][n, h * G + g].double() @ t["prefix_k"][0, h].double().T / math.sqrt(D), scores], 1)
                    all_values = torch.cat([t["prefix_v"][0, h].double(), values])
                w = torch.nan_to_num(torch.softmax(scores, 1))  # a query that sees nothing weighs nothing
                out[n, h * G + g] = (w @ all_values).cpu()
                if weights is not None:
                    weights[n, h, :lens[n]] += w.sum(0).cpu()
    return {"out": out, "weights": weights} if weights is not None else {"out": out}
