"""The decode engine's prompt and sampling operators as measured cases.

Three operators that one request passes through: rotary positions with the append to the
KV cache, attention of a whole prompt (or of single tokens) over that cache, and the draw
of the next token from the logits.  ``own`` false computes them in their plain form with
elementary torch operations; true makes the calls a user of the package makes.

Sizes: 64 query and 8 KV heads of 64 with a 128-token window and a vocabulary of 201088
are the large model's of this repository; the other head shapes and vocabularies are
generic.
"""
import importlib
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}

# the large model's rotary scaling: theta 150000, factor 32 over 4096 positions
_THETA, _FACTOR, _CONTEXT = 150000.0, 32.0, 4096.0


def _ints(text):
    return [int(v) for v in str(text).split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 64 sequences at scattered positions of a long context
        {"name": "rope_step64", "op": "rope", "tokens": 64, "q_heads": 64, "kv_heads": 8,
         "head_dim": 64, "rotary_dim": 64, "interleaved": False, "dtype": "bf16",
         "max_pos": 131072, "skip_every": 9},
        # the rows of one prompt piece, an odd count, into a cache
        {"name": "rope_prompt8191", "op": "rope", "tokens": 8191, "q_heads": 64, "kv_heads": 8,
         "head_dim": 64, "rotary_dim": 64, "interleaved": False, "dtype": "bf16",
         "max_pos": 131072, "skip_every": 0},
        # half of each head rotated, neighbouring pairs, another 16-bit type
        {"name": "rope_partial_pairs", "op": "rope", "tokens": 30011, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "rotary_dim": 64, "interleaved": True, "dtype": "fp16",
         "max_pos": 32768, "skip_every": 0},
        # a whole prompt of one sequence, full causal layer with sinks
        {"name": "attn_prompt8192", "op": "attention", "q_lens": "8192", "kv_lens": "8192",
         "q_heads": 64, "kv_heads": 8, "head_dim": 64, "window": 0, "sinks": True,
         "dtype": "bf16"},
        # prompts of different lengths packed in one call, sliding-window layer
        {"name": "attn_packed_window", "op": "attention",
         "q_lens": "1,17,129,500,1023,2047,4099,33,5000,777",
         "kv_lens": "1,17,129,500,1023,2047,4099,33,5000,777",
         "q_heads": 64, "kv_heads": 8, "head_dim": 64, "window": 128, "sinks": True,
         "dtype": "bf16"},
        # prompt pieces on contexts already in the cache, 128-wide heads, no sinks
        {"name": "attn_pieces_d128", "op": "attention", "q_lens": "511,2049,130,1000",
         "kv_lens": "8703,4097,16130,1000", "q_heads": 32, "kv_heads": 4, "head_dim": 128,
         "window": 0, "sinks": False, "dtype": "fp16"},
        # a decode step: one token each of 64 sequences of different lengths
        {"name": "attn_tokens64", "op": "attention", "q_lens": _text([1] * 64),
         "kv_lens": _text([1 + (i * 1237) % 8000 for i in range(64)]),
         "q_heads": 64, "kv_heads": 8, "head_dim": 64, "window": 0, "sinks": True,
         "dtype": "bf16"},
        # one token of one sequence at the end of a long context
        {"name": "attn_token_long", "op": "attention", "q_lens": "1", "kv_lens": "131071",
         "q_heads": 64, "kv_heads": 8, "head_dim": 64, "window": 0, "sinks": True,
         "dtype": "bf16"},
        # one user's next token, all filters
        {"name": "sample_row", "op": "sample", "rows": 1, "vocab": 201088, "dtype": "fp32",
         "filters": "all"},
        # a serving batch in which every row has its own settings, greedy rows among them
        {"name": "sample_mixed64", "op": "sample", "rows": 64, "vocab": 201088, "dtype": "fp32",
         "filters": "mixed"},
        # a large batch drawn with a temperature only
        {"name": "sample_temperature512", "op": "sample", "rows": 512, "vocab": 201088,
         "dtype": "fp32", "filters": "temperature"},
        # a smaller vocabulary of odd size, 16-bit logits, nucleus sampling
        {"name": "sample_nucleus_odd", "op": "sample", "rows": 96, "vocab": 50257,
         "dtype": "bf16", "filters": "nucleus"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "sample"])
    if op == "rope":
        head_dim = rng.choice([32, 64, 128])
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 6, 8])
        rotary = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4 * 3])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        room = 30011 * 40 * 128 * 2 // (kv * (group + 2) * head_dim * _SIZES[dtype])
        return {"op": "rope", "tokens": _log_int(rng, 1, min(room, 60000)), "q_heads": kv * group,
                "kv_heads": kv, "head_dim": head_dim, "rotary_dim": rotary,
                "interleaved": rng.random() < 0.4, "dtype": dtype,
                "max_pos": _log_int(rng, 512, 1 << 20), "skip_every": rng.choice([0, 0, 7])}
    if op == "attention":
        head_dim = rng.choice([32, 64, 64, 128])
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 7, 8, 8])
        window = rng.choice([0, 0, 128, _log_int(rng, 1, 2000)])
        budget = 4 * 64 * 64 * 8192 * 4096  # the largest listed case's operations
        q_lens, kv_lens, spent = [], [], 0.0
        for _ in range(_log_int(rng, 1, 64)):
            q = 1 if rng.random() < 0.4 else _log_int(rng, 1, 6000)
            ctx = rng.choice([0, 0, _log_int(rng, 1, 20000)])
            cost = 4.0 * head_dim * kv * group * q * (ctx + q / 2 + 1)
            if q_lens and spent + cost > budget or sum(kv_lens) + q + ctx > 131072:
                continue
            q_lens.append(q)
            kv_lens.append(q + ctx)
            spent += cost
        return {"op": "attention", "q_lens": _text(q_lens), "kv_lens": _text(kv_lens),
                "q_heads": kv * group, "kv_heads": kv, "head_dim": head_dim, "window": window,
                "sinks": rng.random() < 0.6, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    vocab = rng.choice([201088, 50257, _log_int(rng, 1000, 201088)])
    rows = _log_int(rng, 1, max(1, min(2000, 512 * 201088 // vocab)))
    return {"op": "sample", "rows": rows, "vocab": vocab,
            "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
            "filters": rng.choice(["all", "mixed", "temperature", "nucleus", "top_k"])}


# ------------------------------------------------------------------------------ inputs
def _inv_freq(rotary_dim):
    """Rotary frequencies in fp32, interpolated for long contexts (YaRN, betas 32 and 1),
    and the factor on cosine and sine that goes with them."""
    half = rotary_dim // 2
    freq = _THETA ** (np.arange(half, dtype=np.float64) * 2 / rotary_dim)
    low = half * math.log(_CONTEXT / (32.0 * 2 * math.pi)) / math.log(_THETA)
    high = half * math.log(_CONTEXT / (1.0 * 2 * math.pi)) / math.log(_THETA)
    ramp = np.clip((np.arange(half) - low) / (high - low), 0, 1)
    inv = ramp / (_FACTOR * freq) + (1 - ramp) / freq
    return inv.astype(np.float32), float(np.float32(0.1 * math.log(_FACTOR) + 1.0))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 13)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * std

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=dev, dtype=torch.float32)

    st = {"case": case}
    if own:
        st["pkg"] = importlib.import_module("gpt-oss_b200")
    if case["op"] == "rope":
        t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        # one projection output per token, q | k | v, as the projection leaves it
        st["qkv"] = normal(t, (hq + 2 * hkv) * d).to(dtype)
        pos = torch.randint(0, case["max_pos"], (t,), generator=gen, device=dev, dtype=torch.int32)
        if case["skip_every"]:  # rows of the batch that hold no sequence now
            pos[case["skip_every"] - 1::case["skip_every"]] = -1
        st["pos"] = pos
        n_slots = t + 61
        st["slots"] = torch.randperm(n_slots, generator=gen, device=dev)[:t].to(torch.int64)
        inv, st["concentration"] = _inv_freq(case["rotary_dim"])
        st["inv_freq"] = torch.from_numpy(inv).to(dev)
        st["q_out"] = torch.zeros(t, hq, d, device=dev, dtype=dtype)
        st["k_cache"] = torch.zeros(n_slots, hkv, d, device=dev, dtype=dtype)
        st["v_cache"] = torch.zeros(n_slots, hkv, d, device=dev, dtype=dtype)
    elif case["op"] == "attention":
        hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        q_lens, kv_lens = _ints(case["q_lens"]), _ints(case["kv_lens"])
        st["q_lens"], st["kv_lens"] = q_lens, kv_lens
        # cache rows: sequences one after the other with unused rows between them
        starts, at = [], 3
        for n in kv_lens:
            starts.append(at)
            at += n + 5
        st["q"] = normal(sum(q_lens), hq, d).to(dtype)
        st["k"] = normal(at, hkv, d).to(dtype)
        st["v"] = normal(at, hkv, d).to(dtype)
        st["starts"] = starts
        st["sinks"] = normal(hq) if case["sinks"] else None
        st["q_start"] = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32,
                                     device=dev)
        st["kv_start"] = torch.tensor(starts, dtype=torch.int64, device=dev)
        st["kv_len"] = torch.tensor(kv_lens, dtype=torch.int32, device=dev)
        st["scale"] = 1.0 / math.sqrt(d)
        st["out"] = torch.zeros_like(st["q"])
    else:
        n, vocab, filters = case["rows"], case["vocab"], case["filters"]
        logits = normal(n, vocab, std=2.0)
        # a few likely continuations stand out of the bulk
        likely = torch.randint(0, vocab, (n, 24), generator=gen, device=dev)
        logits.scatter_add_(1, likely, 10.0 * uniform(n, 24))
        st["logits"] = logits.to(dtype)
        st["u"] = uniform(n)
        st["temperature"] = 0.6 + 0.7 * uniform(n)
        top_k = torch.randint(20, 200, (n,), generator=gen, device=dev, dtype=torch.int32)
        top_p = 0.8 + 0.19 * uniform(n)
        min_p = 0.02 + 0.08 * uniform(n)
        kind = torch.randint(0, 5, (n,), generator=gen, device=dev)
        if filters == "mixed":
            # greedy, all filters, top-k only, top-p only, temperature only
            st["temperature"] = torch.where(kind == 0, 0.0, st["temperature"])
            st["top_k"] = torch.where((kind == 1) | (kind == 2), top_k, 0)
            st["top_p"] = torch.where((kind == 1) | (kind == 3), top_p, 1.0)
            st["min_p"] = torch.where(kind == 1, min_p, 0.0)
        else:
            st["top_k"] = top_k if filters in ("all", "top_k") else None
            st["top_p"] = top_p if filters in ("all", "nucleus") else None
            st["min_p"] = min_p if filters == "all" else None
        st["next"] = torch.zeros(n, dtype=torch.int32, device=dev)
    return st


# -------------------------------------------------------------------------- plain forms
def _rope_plain(st):
    case = st["case"]
    t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    r = case["rotary_dim"]
    x = st["qkv"].view(t, hq + 2 * hkv, d).float()
    ang = st["pos"].double()[:, None] * st["inv_freq"].double()[None, :]
    cos = (torch.cos(ang).float() * st["concentration"])[:, None, :]
    sin = (torch.sin(ang).float() * st["concentration"])[:, None, :]
    qk = x[:, :hq + hkv]
    if case["interleaved"]:
        a, b = qk[..., 0:r:2], qk[..., 1:r:2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = qk[..., :r // 2], qk[..., r // 2:r]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qk = torch.cat([rot, qk[..., r:]], -1).to(st["qkv"].dtype)
    live = st["pos"] >= 0
    st["q_out"][live] = qk[live, :hq]
    slots = st["slots"][live]
    st["k_cache"][slots] = qk[live, hq:]
    st["v_cache"][slots] = st["qkv"].view(t, hq + 2 * hkv, d)[live, hq + hkv:]
    return [st["q_out"], st["k_cache"], st["v_cache"]]


def _attention_plain(st):
    case = st["case"]
    hkv, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    d, window = case["head_dim"], case["window"]
    at = 0
    for q_len, kv_len, start in zip(st["q_lens"], st["kv_lens"], st["starts"]):
        k = st["k"][start:start + kv_len].float()
        v = st["v"][start:start + kv_len].float()
        step = max(1, min(q_len, (1 << 29) // (kv_len * group)))
        for q0 in range(0, q_len, step):
            n = min(step, q_len - q0)
            pos = torch.arange(q0, q0 + n, device=k.device) + (kv_len - q_len)
            first = max(0, kv_len - q_len + q0 - window + 1) if window else 0
            last = kv_len - q_len + q0 + n
            t = torch.arange(first, last, device=k.device)
            hidden = t[None, :] > pos[:, None]
            if window:
                hidden = hidden | (t[None, :] <= pos[:, None] - window)
            for h in range(hkv):
                rows = slice(at + q0, at + q0 + n)
                heads = slice(h * group, (h + 1) * group)
                q = st["q"][rows, heads].float().transpose(0, 1).reshape(group * n, d)
                s = (q @ k[first:last, h].T * st["scale"]).view(group, n, -1)
                s = s.masked_fill(hidden, -math.inf)
                m = s.amax(-1, keepdim=True)
                if st["sinks"] is not None:
                    sink = st["sinks"][heads].view(group, 1, 1)
                    m = torch.maximum(m, sink)
                e = torch.exp(s - m)
                z = e.sum(-1, keepdim=True)
                if st["sinks"] is not None:
                    z = z + torch.exp(sink - m)
                o = (e.view(group * n, -1) @ v[first:last, h]).view(group, n, d) / z
                st["out"][rows, heads] = o.transpose(0, 1).to(st["out"].dtype)
        at += q_len
    return st["out"]


def _sample_plain(st):
    logits = st["logits"].double()
    n, vocab = logits.shape
    out = st["next"]
    for r0 in range(0, n, 64):
        x = logits[r0:r0 + 64]
        rows = slice(r0, r0 + x.shape[0])
        greedy = st["temperature"][rows] <= 0
        temp = torch.where(greedy, 1.0, st["temperature"][rows]).double()[:, None]
        value, order = torch.sort(x, dim=1, descending=True, stable=True)
        w = torch.exp((value - value[:, :1]) / temp)
        rank = torch.arange(vocab, device=x.device)[None, :]
        keep = torch.ones_like(w, dtype=torch.bool)
        if st["top_k"] is not None:
            k = st["top_k"][rows].long()[:, None]
            keep &= (rank < k) | (k <= 0)
        if st["top_p"] is not None:
            p = st["top_p"][rows].double()[:, None]
            kept = torch.where(keep, w, 0.0)
            before = torch.cumsum(kept, 1) - kept
            keep &= (before < p * kept.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)
        if st["min_p"] is not None:
            keep &= w >= st["min_p"][rows].double()[:, None]
        mass = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
        cum = torch.cumsum(mass, 1)
        target = st["u"][rows].double()[:, None] * cum[:, -1:]
        index = torch.arange(vocab, device=x.device)[None, :]
        pick = torch.where((cum > target) & (mass > 0), index, vocab).amin(1)
        out[rows] = torch.where(greedy, order[:, 0], pick).to(torch.int32)
    return out


# ------------------------------------------------------------------------------- a pass
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"rope": _rope_plain, "attention": _attention_plain,
                "sample": _sample_plain}[op](state)
    case, pkg = state["case"], state["pkg"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "rope":
        hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        qkv = state["qkv"].view(case["tokens"], hq + 2 * hkv, d)
        pkg.rope_append(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], state["pos"],
                        state["inv_freq"], state["q_out"], state["k_cache"], state["v_cache"],
                        slots=state["slots"], concentration=state["concentration"],
                        interleaved=case["interleaved"], stream=stream)
        return [state["q_out"], state["k_cache"], state["v_cache"]]
    if op == "attention":
        pkg.prompt_attention(state["q"], state["k"], state["v"], state["q_start"],
                             state["kv_start"], state["kv_len"], state["out"],
                             sinks=state["sinks"], scale=state["scale"], window=case["window"],
                             max_kv_len=max(state["kv_lens"]), stream=stream)
        return state["out"]
    pkg.sample_tokens(state["logits"], state["u"], state["next"],
                      temperature=state["temperature"], top_k=state["top_k"],
                      top_p=state["top_p"], min_p=state["min_p"], stream=stream)
    return state["next"]


# --------------------------------------------------------------------------------- work
def _visible(q_len, kv_len, window):
    """Pairs of query and visible key, and keys that any query sees."""
    pos = np.arange(kv_len - q_len, kv_len, dtype=np.int64)
    seen = pos + 1
    if window:
        seen = np.minimum(seen, window)
    keys = min(kv_len, q_len + window - 1) if window else kv_len
    return int(seen.sum()), keys


def work(case):
    size = _SIZES[case["dtype"]]
    if case["op"] == "rope":
        t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        live = t - (t // case["skip_every"] if case["skip_every"] else 0)
        return {"bytes": 2 * live * (hq + 2 * hkv) * d * size + t * 12,
                "flops": 3 * live * (hq + hkv) * case["rotary_dim"]}
    if case["op"] == "attention":
        hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        pairs = keys = tokens = 0
        for q_len, kv_len in zip(_ints(case["q_lens"]), _ints(case["kv_lens"])):
            p, k = _visible(q_len, kv_len, case["window"])
            pairs, keys, tokens = pairs + p, keys + k, tokens + q_len
        return {"bytes": (2 * tokens * hq + 2 * keys * hkv) * d * size,
                "flops": 4 * pairs * hq * d}
    n, vocab = case["rows"], case["vocab"]
    return {"bytes": n * vocab * size + 24 * n, "flops": 4 * n * vocab}


# ------------------------------------------------------------------------------ oracles
def _rope_exact(case, st):
    t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    half = case["rotary_dim"] // 2
    rows = st["qkv"].double().reshape(t, hq + 2 * hkv, d)
    live = torch.nonzero(st["pos"] >= 0).flatten()
    out = rows[live].clone()
    phase = torch.polar(torch.full((1, 1), st["concentration"], dtype=torch.float64,
                                   device=rows.device),
                        st["pos"][live].double()[:, None] * st["inv_freq"].double())
    if case["interleaved"]:
        first = torch.arange(half, device=rows.device) * 2
        second = first + 1
    else:
        first = torch.arange(half, device=rows.device)
        second = first + half
    for h in range(hq + hkv):
        turned = torch.complex(out[:, h, first], out[:, h, second]) * phase
        out[:, h, first], out[:, h, second] = turned.real, turned.imag
    res = [torch.zeros(st["q_out"].shape, dtype=torch.float64, device=rows.device),
           torch.zeros(st["k_cache"].shape, dtype=torch.float64, device=rows.device),
           torch.zeros(st["v_cache"].shape, dtype=torch.float64, device=rows.device)]
    res[0].index_copy_(0, live, out[:, :hq])
    res[1].index_copy_(0, st["slots"][live], out[:, hq:hq + hkv])
    res[2].index_copy_(0, st["slots"][live], out[:, hq + hkv:])
    return res


def _attention_exact(case, st):
    hq, hkv, d, window = case["q_heads"], case["kv_heads"], case["head_dim"], case["window"]
    group = hq // hkv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    row = 0
    for q_len, kv_len, start in zip(st["q_lens"], st["kv_lens"], st["starts"]):
        offset = kv_len - q_len
        for h in range(hq):
            key = st["k"][start:start + kv_len, h // group].double()
            val = st["v"][start:start + kv_len, h // group].double()
            for q0 in range(0, q_len, 1024):
                q1 = min(q0 + 1024, q_len)
                lo = max(0, offset + q0 + 1 - window) if window else 0
                hi = offset + q1
                z = torch.einsum("qd,kd->qk", st["q"][row + q0:row + q1, h].double(), key[lo:hi])
                z = z * st["scale"]
                delta = (torch.arange(q0, q1, device=z.device)[:, None] + offset
                         - torch.arange(lo, hi, device=z.device)[None, :])
                seen = (delta >= 0) & (delta < window) if window else delta >= 0
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                if st["sinks"] is not None:
                    z = torch.cat([z, st["sinks"][h].double().expand(q1 - q0, 1)], 1)
                p = torch.softmax(z, 1)[:, :hi - lo]
                out[row + q0:row + q1, h] = p @ val[lo:hi]
        row += q_len
    return out


def _sample_exact(case, st):
    settings = {k: None if st[k] is None else st[k].double().cpu().numpy()
                for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    picks = np.zeros(case["rows"], dtype=np.int32)
    for r in range(case["rows"]):
        x = st["logits"][r].double()
        best = x.max()
        if settings["temperature"][r] <= 0:
            picks[r] = int(torch.nonzero(x == best)[0])
            continue
        # the kept ids, likeliest first until the last step puts them back in their order
        ids = torch.arange(x.numel(), device=x.device)
        k = 0 if settings["top_k"] is None else int(settings["top_k"][r])
        p = 1.0 if settings["top_p"] is None else settings["top_p"][r]
        if 0 < k < x.numel():
            ids = torch.nonzero(x >= torch.topk(x, k).values[-1]).flatten()
        if k > 0 or p < 1:
            ids = ids[torch.argsort(-x[ids], stable=True)]
        if 0 < k < x.numel():
            ids = ids[:k]
        w = torch.exp((x[ids] - best) / settings["temperature"][r])
        if p < 1:
            total = torch.cumsum(w, 0)
            n = 1 + int(torch.searchsorted(total[:-1], p * total[-1], side="left"))
            ids, w = ids[:n], w[:n]
        if settings["min_p"] is not None:
            ids = ids[w >= settings["min_p"][r]]
        ids = torch.sort(ids).values
        total = torch.cumsum(torch.exp((x[ids] - best) / settings["temperature"][r]), 0)
        at = int(torch.searchsorted(total, settings["u"][r] * total[-1], side="right"))
        picks[r] = int(ids[min(at, ids.numel() - 1)])
    return torch.from_numpy(picks)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _rope_exact(case, st)
    if case["op"] == "attention":
        if work(case)["flops"] > 2e12:
            return None
        return _attention_exact(case, st)
    return _sample_exact(case, st)
