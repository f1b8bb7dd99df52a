"""Performance cases of answering several times from one prompt, one operator a pass.

* ``dense``   attention of decode rows or of a chunk's rows over every cached key, with scores capped
  by a tanh, a bias that falls with the distance, or a sliding window (``ops.dense_attention_kvcache``);
* ``shared``  attention of a batch whose sequences begin with one long prefix, kept once, and go on
  in caches of their own (``ops.shared_prefix_attention``);
* ``sample``  the next token of each row from its logits and a given random number, with
  temperature, top-k, top-p and min-p (``ops.sample_logits``).

A row of a sequence with ``n`` query rows and ``len`` keys (prefix included) that is its ``i``-th stands
at position ``p = len - n + i``.  Key ``j`` is visible where ``j < len``, with ``causal`` ``j <= p`` and
with a window ``j >= p - left``.  Its score is ``x = scale q.k``, then ``cap tanh(x / cap)``, then less
``slope_h |p - j|``.

A token's weight is ``exp((x - max x) / temperature)``.  Ordered by logit, ties to the lower index,
the first ``top_k`` are kept, of these the shortest run whose weights reach ``top_p`` of their sum, of
these those of at least ``min_p`` of the largest; the draw is the lowest index at which the running
sum of the kept weights, in the vocabulary's order, exceeds ``u`` times their sum.

Sizes are those of the MiniCPM4.1-8B shape (32 query and 2 KV heads of 128, vocabulary 73448); the
drawn cases add other head counts and odd sizes.
"""
import math

import torch

own = False

DEV = "cuda"
D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LENS_16 = "2047,2500,3333,4095,5000,6144,8191,9999,12287,16000,20001,24576,32767,40000,50001,65535"


def listed():
    return [
        # One decode step of a 128K conversation in a layer with a sliding window.
        _dense("window_128k_b1", "131071", "1", window=4095),
        # One decode step of sixteen conversations in a layer with capped scores.
        _dense("softcap_ragged_b16", LENS_16, ",".join(["1"] * 16), cap=50.0),
        # One decode step of eight conversations with a bias by distance, eight KV heads, in fp16.
        _dense("alibi_ragged_b8_fp16", "1,517,4097,9001,16383,12000,8191,2048", "1,1,1,1,1,1,1,1",
               alibi=True, G=8, dtype="fp16"),
        # A later chunk of a prompt: 1024 tokens behind 32K.
        _dense("softcap_chunk_1k", "33791", "1024", cap=30.0, causal=True),
        # Two prompts into empty caches, in fp16, with a bias by distance and a window.
        _dense("alibi_prompts_fp16", "4096,1337", "4096,1337", alibi=True, window=2000, causal=True,
               dtype="fp16"),
        # Four answers to a 32K prompt, 1 to 200 tokens each.
        _shared("shared_32k_b4_fp16", 32768, "1,200,77,130", "1,1,1,1", dtype="fp16"),
        # Sixteen answers to a 128K prompt.
        _shared("shared_128k_b16", 131072, "1,33,64,100,129,200,256,300,333,400,444,500,512,600,640,700",
                ",".join(["1"] * 16)),
        # Sixty-four answers to a 64K prompt.
        _shared("shared_64k_b64", 65000, ",".join(str(1 + 31 * i) for i in range(64)),
                ",".join(["1"] * 64)),
        # Eight answers whose next four tokens were guessed, with capped scores and a window.
        _shared("shared_guessed_b8", 9001, "4,40,100,300,517,777,1000,1337", "4,4,4,4,4,4,4,4", cap=50.0,
                window=8191, causal=True),
        # The next token of one answer.
        _sample("sample_b1", 1, temperature=0.8, top_k=50, top_p=0.9),
        # The next tokens of sixteen, from logits in 16 bits, without a top-k.
        _sample("sample_b16_bf16", 16, temperature=0.7, top_p=0.95, min_p=0.01, dtype="bf16"),
        # The next tokens of a served batch whose requests set their own temperature and cuts.
        _sample("sample_b256_mixed", 256, mixed=True),
    ]


def _dense(name, lens, new, *, cap=0.0, alibi=False, window=-1, causal=False, H=32, G=2, dtype="bf16"):
    return dict(name=name, kind="dense", lens=lens, new=new, cap=cap, alibi=alibi, window=window,
                causal=causal, H=H, G=G, dtype=dtype)


def _shared(name, prefix, lens, new, *, cap=0.0, alibi=False, window=-1, causal=False, H=32, G=2,
            dtype="bf16"):
    return dict(name=name, kind="shared", prefix=prefix, lens=lens, new=new, cap=cap, alibi=alibi,
                window=window, causal=causal, H=H, G=G, dtype=dtype)


def _sample(name, rows, *, vocab=73448, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False,
            dtype="fp32"):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, temperature=temperature, top_k=top_k,
                top_p=top_p, min_p=min_p, mixed=mixed, dtype=dtype)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(map(str, values))


def draw(rng):
    kind = rng.choice(("dense", "dense", "shared", "shared", "sample"))
    if kind == "sample":
        case = _sample("", _log_int(rng, 1, 256), vocab=_log_int(rng, 300, 73448),
                       temperature=rng.choice((0.0, 0.6, 1.0, 1.3)), top_k=rng.choice((0, 0, 1, 20, 200)),
                       top_p=rng.choice((1.0, 0.5, 0.9, 0.99)), min_p=rng.choice((0.0, 0.0, 0.05)),
                       mixed=rng.random() < 0.3, dtype=rng.choice(("fp32", "bf16", "fp16")))
        del case["name"]
        return case
    H, G = rng.choice(((32, 2), (32, 2), (32, 8), (16, 1), (24, 4), (5, 5)))
    more = dict(cap=rng.choice((0.0, 30.0)), alibi=rng.random() < 0.4, window=rng.choice((-1, _log_int(rng, 1, 9000))),
                H=H, G=G, dtype=rng.choice(("bf16", "bf16", "fp16")))
    if kind == "dense" and rng.random() < 0.3:  # a chunk
        batch = _log_int(rng, 1, 4)
        new = [_log_int(rng, 2, 1024 // batch) for _ in range(batch)]
        lens = [n + _log_int(rng, 1, 30000) for n in new]
        case = _dense("", _text(lens), _text(new), causal=True, **more)
    else:
        rows = rng.choice((1, 1, 1, 3))
        batch = _log_int(rng, 1, 24 if kind == "dense" else 48)
        top = (40000 if G <= 2 else 9000) if kind == "dense" else 1500
        lens = [max(rows, _log_int(rng, 1, top)) for _ in range(batch)]
        new = [rows] * batch
        causal = rows > 1 or rng.random() < 0.5
        if kind == "dense":
            case = _dense("", _text(lens), _text(new), causal=causal, **more)
        else:
            case = _shared("", _log_int(rng, 64, 60000 if G <= 2 else 20000), _text(lens), _text(new),
                           causal=causal, **more)
            if case["window"] >= 0:
                case["window"] += case["prefix"] // 2
    del case["name"]
    return case


def _ints(text):
    return [int(x) for x in text.split(",")]


def _cu(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _keys(shape, gen):
    """Keys with a few strong channels and offsets of their own, as after a rotary embedding."""
    gain = torch.exp(0.5 * torch.randn(shape[-2:], device=DEV, generator=gen))
    gain[..., :4] *= 4.0
    shift = 0.5 * gain * torch.randn(shape[-2:], device=DEV, generator=gen)
    return torch.randn(shape, device=DEV, generator=gen) * gain + shift


def _prepare_attention(case, gen):
    lens, new, H, G = _ints(case["lens"]), _ints(case["new"]), case["H"], case["G"]
    dtype = DTYPES[case["dtype"]]
    capacity = -(-max(lens) // 64) * 64
    shape = (len(lens), capacity, G, D)  # rows past a sequence's end hold what was there before
    st = dict(k=_keys(shape, gen).to(dtype), v=torch.randn(shape, device=DEV, generator=gen).to(dtype),
              q=torch.randn(sum(new), H, D, device=DEV, generator=gen).to(dtype), lens=_i32(lens),
              cu=_i32(_cu(new)), longest=max(lens), most=max(new), causal=case["causal"],
              cap=case["cap"], window=case["window"], slopes=None)
    if case["alibi"]:  # the geometric slopes 2^(-8 (h + 1) / H)
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEV)
    if case["kind"] == "shared":
        shape = (case["prefix"], G, D)
        st["k_prefix"] = _keys(shape, gen).to(dtype)
        st["v_prefix"] = torch.randn(shape, device=DEV, generator=gen).to(dtype)
    return st


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    x = 2.0 * torch.randn(rows, vocab, device=DEV, generator=gen)
    likely = torch.randint(0, vocab, (rows, 40), device=DEV, generator=gen)  # what the context asks for
    x.scatter_add_(1, likely, 6.0 + 3.0 * torch.randn(rows, 40, device=DEV, generator=gen))
    dtype = DTYPES[case["dtype"]]
    if dtype is torch.float32:  # a 16-bit head's logits, as the model gives them
        x = x.to(torch.bfloat16)
    st = dict(logits=x.to(dtype), u=torch.rand(rows, device=DEV, generator=gen))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        st[name] = case[name]
    if case["mixed"]:
        def pick(values, dtype=torch.float32):
            at = torch.randint(0, len(values), (rows,), device=DEV, generator=gen)
            return torch.tensor(values, dtype=dtype, device=DEV)[at]
        st.update(temperature=pick((0.0, 0.5, 0.8, 1.0, 1.5)), top_k=pick((0, 1, 40, 100, 1000), torch.int32),
                  top_p=pick((0.3, 0.8, 0.95, 1.0)), min_p=pick((0.0, 0.0, 0.02, 0.2)))
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = (_prepare_sample if case["kind"] == "sample" else _prepare_attention)(case, gen)
    return dict(st, kind=case["kind"])


# ---------------------------------------------------------------------------
# One pass: the plain forms
# ---------------------------------------------------------------------------
def _scores(x, pos, at, seen, st, G):
    """Scores of ``x [.., G, heads, rows, keys]`` (products, unscaled) of rows at ``pos`` and keys at ``at``."""
    x = x * D ** -0.5
    if st["cap"] > 0:
        x = st["cap"] * torch.tanh(x / st["cap"])
    far = pos[..., :, None] - at
    if st["slopes"] is not None:
        x = x - st["slopes"].view(G, -1, 1, 1) * far.abs()[..., None, None, :, :]
    if st["causal"]:
        seen = seen & (far >= 0)
    if st["window"] >= 0:
        seen = seen & (far <= st["window"])
    return x.masked_fill(~seen[..., None, None, :, :], float("-inf"))


def _attention_plain(st):
    q, k, v = st["q"].float(), st["k"][:, :st["longest"]].float(), st["v"][:, :st["longest"]].float()
    total, H, _ = q.shape
    G, most = k.shape[2], st["most"]
    lens, cu = st["lens"].long(), st["cu"].long()
    n = cu[1:] - cu[:-1]
    before = st["k_prefix"].shape[0] if "k_prefix" in st else 0
    # Rows padded to [batch, most], behind their sequence's end.
    row = torch.arange(most, device=DEV)
    held = row < n[:, None]
    x = q[(cu[:-1, None] + row).clamp(max=total - 1)]  # [batch, most, H, D]
    x = x.view(*x.shape[:2], G, H // G, D).permute(0, 2, 3, 1, 4)  # [batch, G, heads, most, D]
    pos = before + (lens - n)[:, None] + row
    at = torch.arange(k.shape[1], device=DEV)
    keys = k.permute(0, 2, 3, 1).unsqueeze(2)  # [batch, G, 1, D, keys]
    s = _scores(x @ keys, pos, before + at, (at < lens[:, None])[:, None, :], st, G)
    if before:
        kp, vp = st["k_prefix"].float(), st["v_prefix"].float()
        flat = q.view(total, G, H // G, D).permute(1, 2, 0, 3)  # [G, heads, rows, D]
        first = torch.arange(before, device=DEV)
        here = pos[held]  # the packed rows' positions
        seen = torch.ones(1, before, dtype=torch.bool, device=DEV)
        sp = _scores(flat @ kp.permute(1, 2, 0).unsqueeze(1), here, first, seen, st, G)
        top = sp.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), 0.0, top)
        pp = torch.exp(sp - top)
        sum_p, out_p = pp.sum(-1), pp @ vp.transpose(0, 1).unsqueeze(1)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(s - m)
    out = p @ v.transpose(1, 2).unsqueeze(2)  # [batch, G, heads, most, D]
    l = p.sum(-1)
    out, l, m = (t.movedim(3, 1)[held] for t in (out, l, m.squeeze(-1)))  # [rows, G, heads(, D)]
    if before:
        out_p, sum_p, top = (t.movedim(2, 0) for t in (out_p, sum_p, top.squeeze(-1)))
        both = torch.maximum(torch.where(l > 0, m, top), torch.where(sum_p > 0, top, m))
        a, b = torch.exp(m - both) * (l > 0), torch.exp(top - both) * (sum_p > 0)
        out = out * a[..., None] + out_p * b[..., None]
        l, m = l * a + sum_p * b, both
    out = (out / l[..., None]).reshape(total, H, D).to(st["q"].dtype)
    return out, (m + torch.log(l)).reshape(total, H).t().contiguous()


def _column(value, rows):
    """A setting of the batch, or one of each row, as float64 ``[rows, 1]``."""
    if torch.is_tensor(value):
        return value.double()[:, None]
    return torch.full((rows, 1), float(value), dtype=torch.float64, device=DEV)


def _sample_plain(st):
    x = st["logits"].double()
    rows, vocab = x.shape
    t, k, p, least = (_column(st[n], rows) for n in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device=DEV)
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    w = torch.where((t > 0) | (rank == 0), w, 0.0)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(-1) - w
    w = torch.where((p >= 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0), w, 0.0)
    w = torch.where(w >= least, w, 0.0)
    w = torch.empty_like(w).scatter_(1, order, w)  # back in the vocabulary's order
    upto = w.cumsum(-1)
    total = upto[:, -1:]
    token = (upto <= st["u"].double()[:, None] * total).sum(-1, keepdim=True)
    token = token.clamp(max=vocab - 1)
    logprob = torch.log(w.gather(1, token) / total)
    return token[:, 0].to(torch.int32), logprob[:, 0].float()


def _run_own(st):
    from leanselect_amd import ops

    if st["kind"] == "sample":
        return ops.sample_logits(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                 top_p=st["top_p"], min_p=st["min_p"], return_logprob=True)
    more = dict(causal=st["causal"], softcap=st["cap"], alibi_slopes=st["slopes"],
                window=(st["window"], -1), return_lse=True)
    if st["kind"] == "shared":
        return ops.shared_prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"],
                                           st["lens"], st["cu"], st["longest"], **more)
    return ops.dense_attention_kvcache(st["q"], st["k"], st["v"], st["lens"], st["cu"], st["longest"],
                                       **more)


def run(state):
    if own:
        return _run_own(state)
    return _sample_plain(state) if state["kind"] == "sample" else _attention_plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4.0 if case["dtype"] == "fp32" else 2.0), "flops": 4.0 * n}
    before = case.get("prefix", 0)
    H, G, left = case["H"], case["G"], case["window"]
    pairs = keys = 0
    first_prefix = before
    for length, n in zip(_ints(case["lens"]), _ints(case["new"])):
        end = before + length
        first = max(0, end - n - left) if left >= 0 else 0
        keys += end - max(first, before)
        first_prefix = min(first_prefix, first)
        for i in range(n):
            p = end - n + i
            low = max(0, p - left) if left >= 0 else 0
            pairs += (p + 1 if case["causal"] else end) - low
    keys += before - first_prefix
    rows = sum(_ints(case["new"]))
    return {"bytes": 4.0 * keys * G * D + 4.0 * rows * H * D + 4.0 * rows * H, "flops": 4.0 * pairs * H * D}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_attention(case, seed):
    st = prepare(case, seed)
    q = st["q"].double()
    total, H, _ = q.shape
    G, before = case["G"], case.get("prefix", 0)
    heads = H // G
    out, lse = torch.zeros_like(q), torch.zeros(H, total, dtype=torch.float64, device=DEV)
    at = 0
    for b, (length, n) in enumerate(zip(_ints(case["lens"]), _ints(case["new"]))):
        j = torch.arange(before + length, device=DEV)
        for g in range(G):
            k, v = st["k"][b, :length, g].double(), st["v"][b, :length, g].double()
            if before:
                k = torch.cat((st["k_prefix"][:, g].double(), k))
                v = torch.cat((st["v_prefix"][:, g].double(), v))
            for i in range(0, n, 128):
                i1 = min(i + 128, n)
                p = torch.arange(before + length - n + i, before + length - n + i1, device=DEV)
                hidden = torch.zeros(i1 - i, j.numel(), dtype=torch.bool, device=DEV)
                if case["causal"]:
                    hidden |= j > p[:, None]
                if case["window"] >= 0:
                    hidden |= j < p[:, None] - case["window"]
                for h in range(g * heads, (g + 1) * heads):
                    x = q[at + i:at + i1, h] @ k.t() / math.sqrt(D)
                    if case["cap"] > 0:
                        x = torch.tanh(x / case["cap"]) * case["cap"]
                    if case["alibi"]:
                        slope = float(st["slopes"][h])
                        x -= slope * (j - p[:, None]).abs().double()
                    x[hidden] = -math.inf
                    lse[h, at + i:at + i1] = torch.logsumexp(x, -1)
                    out[at + i:at + i1, h] = torch.softmax(x, -1) @ v
        at += n
    return out, lse


def _exact_sample(case, seed):
    st = prepare(case, seed)
    x = st["logits"].double().cpu().numpy()
    import numpy as np

    u = st["u"].double().cpu().numpy()
    each = {}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        value = st[name]
        each[name] = value.double().cpu().tolist() if torch.is_tensor(value) else [float(value)] * len(x)
    tokens, logprobs = [], []
    for r, row in enumerate(x):
        t, k = each["temperature"][r], int(each["top_k"][r])
        order = np.lexsort((np.arange(row.size), -row))  # by logit, ties by index
        if t == 0.0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        if k > 0:
            order = order[:k]
        weights = np.exp((row[order] - row[order[0]]) / t)
        if each["top_p"][r] < 1.0:
            n = 1 + np.searchsorted(np.cumsum(weights), each["top_p"][r] * weights.sum(), side="left")
            order, weights = order[:n], weights[:n]
        keep = weights >= each["min_p"][r]
        order, weights = order[keep], weights[keep]
        by_index = np.argsort(order)
        order, weights = order[by_index], weights[by_index]
        upto = np.cumsum(weights)
        i = min(int(np.searchsorted(upto, u[r] * upto[-1], side="right")), order.size - 1)
        tokens.append(int(order[i]))
        logprobs.append(math.log(weights[i] / upto[-1]))
    return (torch.tensor(tokens, dtype=torch.int32, device=DEV),
            torch.tensor(logprobs, dtype=torch.float64, device=DEV))


def exact(case, seed):
    return (_exact_sample if case["kind"] == "sample" else _exact_attention)(case, seed)
