"""Performance cases of decoding in 8 and 4 bits, one operator a pass.

* ``append``  new keys and values into a cache of e4m3 pages with one power-of-two scale for each
  page of 64 tokens and KV head, with the compressed keys they complete (``ops.kvcache_append_q8``);
* ``sparse``  attention of decode rows over the pages of their plans (``ops.sparse_attention_kvcache_q8``);
* ``dense``   the same over every cached page (``ops.dense_attention_kvcache_q8``);
* ``linear``  a product of a few rows with a weight of 4-bit E2M1 values and one power-of-two scale
  for every 32 inputs (``ops.linear_mx4``);
* ``silu``    the gate and up projections of an MLP as one such product, with the gated activation
  (``ops.linear_mx4_silu_mul``).

Cache layout: keys ``[batch, pages, G, 64, 128]`` e4m3; values ``[batch, pages, G, 128, 64]`` e4m3, a
channel's 64 tokens together and token ``16 t + 4 q + i`` at place ``16 q + 4 t + i``; scale codes uint8
``[batch, pages, G]`` of keys and of values, code ``c`` for 2^(c - 127).  Weight layout: see ``_lay_out``.
Sizes are those of the MiniCPM4.1-8B shape (hidden 4096, 32 query and 2 KV heads of 128, MLP 16384,
vocabulary 73448); the drawn cases add other head counts and odd sizes.
"""
import math

import torch

own = False

DEV = "cuda"
D, PAGE = 128, 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # A prompt of 32K tokens into an empty cache, one layer of a prefill.
        dict(name="append_prompt_32k", kind="append", lens="0", new="32768", H=32, G=2, dtype="bf16"),
        # Later chunks of four prompts, from odd lengths: pages begun before and pages left unfinished.
        dict(name="append_chunks_fp16", kind="append", lens="1337,64,4097,0", new="517,1000,2049,33",
             H=32, G=2, dtype="fp16"),
        # One decode step of sixteen conversations.
        dict(name="append_step_b16", kind="append",
             lens="2047,2500,3333,4095,5000,6144,8191,700,1023,33,64,4000,777,2222,5555,7000",
             new="1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1", H=32, G=2, dtype="bf16"),
        # One decode step of a single 128K conversation, 64 pages a group.
        dict(name="sparse_128k_b1", kind="sparse", lens="131071", rows=1, causal=False, budget=64,
             local=4, H=32, G=2, dtype="bf16"),
        # One decode step of a served batch of 16 conversations of 2K to 64K tokens.
        dict(name="sparse_ragged_b16", kind="sparse",
             lens="2047,2500,3333,4095,5000,6144,8191,9999,12287,16000,20001,24576,32767,40000,"
                  "50001,65535",
             rows=1, causal=False, budget=64, local=4, H=32, G=2, dtype="bf16"),
        # A single 128K conversation without a plan.
        dict(name="dense_128k_b1", kind="dense", lens="131071", rows=1, causal=False, H=32, G=2,
             dtype="bf16"),
        # Eight conversations without a plan, as below a model's sparse threshold, in fp16.
        dict(name="dense_ragged_b8_fp16", kind="dense",
             lens="1,517,4097,9001,16383,30000,8191,24001", rows=1, causal=False, H=32, G=2,
             dtype="fp16"),
        # The q/k/v projection of one token.
        dict(name="linear_qkv_b1", kind="linear", rows=1, out=4608, inp=4096, dtype="bf16"),
        # The MLP's down projection of seven tokens, in fp16.
        dict(name="linear_down_b7_fp16", kind="linear", rows=7, out=4096, inp=16384, dtype="fp16"),
        # The head of a batch of 16.
        dict(name="linear_head_b16", kind="linear", rows=16, out=73448, inp=4096, dtype="bf16"),
        # The MLP's gate and up projections of one token.
        dict(name="silu_b1", kind="silu", rows=1, out=32768, inp=4096, dtype="bf16"),
        # The same for a batch of 33.
        dict(name="silu_b33", kind="silu", rows=33, out=32768, inp=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "append", "sparse", "sparse", "dense", "linear", "linear", "silu"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    H, G = rng.choice(((32, 2), (32, 2), (32, 8), (16, 1), (24, 4), (5, 5)))
    if kind == "append":
        batch = _log_int(rng, 1, 24)
        step = rng.random() < 0.5
        total = _log_int(rng, batch, 24000 * 2 // max(2, G))
        lens = [rng.choice((0, _log_int(rng, 1, 6000))) for _ in range(batch)]
        cuts = sorted(rng.random() for _ in range(batch - 1))
        new = [rng.choice((0, 1, 1, 1, 2)) if step else int(total * (b - a))
               for a, b in zip([0.0] + cuts, cuts + [1.0])]
        new[rng.randrange(batch)] += 1
        return dict(kind=kind, lens=",".join(map(str, lens)), new=",".join(map(str, new)), H=H, G=G,
                    dtype=dtype)
    if kind in ("sparse", "dense"):
        rows = rng.choice((1, 1, 1, 3))
        batch = _log_int(rng, 1, 24 if kind == "sparse" else 12)
        top = 131000 if kind == "sparse" and batch <= 4 and G <= 2 else 40000 if G <= 2 else 9000
        lens = [max(rows, _log_int(rng, 3, top)) for _ in range(batch)]
        case = dict(kind=kind, lens=",".join(map(str, lens)), rows=rows,
                    causal=rows > 1 or rng.random() < 0.5, H=H, G=G, dtype=dtype)
        if kind == "sparse":
            budget, local = rng.choice(((64, 4), (96, 32), (17, 3)))
            case.update(budget=budget, local=local)
        return case
    rows = _log_int(rng, 1, 64)
    inp = 8 * _log_int(rng, 16, 2048)
    out = _log_int(rng, 200, 40000)
    if kind == "silu":
        out = 32 * max(8, out // 32)
    return dict(kind=kind, rows=rows, out=out, inp=inp, dtype=dtype)


def _ints(text):
    return [int(x) for x in text.split(",")]


def _cu(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _n_windows(n):
    return (n - 32) // 16 + 1 if n >= 32 else 0


# ---------------------------------------------------------------------------
# The formats
# ---------------------------------------------------------------------------
def _code(top, lead, full, low):
    """Scale code of a set with largest magnitude ``top`` (float32): the least c with
    top <= L 2^(c - 127), L = (1 + full / 2^23) 2^lead the format's largest value."""
    bits = top.contiguous().view(torch.int32)
    return ((bits >> 23) - lead + ((bits & 0x7FFFFF) > full).int()).clamp(low, 254)


def _e4m3_code(top):
    return _code(top, 8, 0x600000, 1)  # 448 = 1.75 2^8


def _power(code):
    """2^(code - 127) as float32, of codes 1 to 254."""
    return (code.int() << 23).view(torch.float32)


def _place(token):
    """Where a page's value of this token is kept among its channel's 64."""
    return ((token >> 2) & 3) * 16 + (token >> 4) * 4 + (token & 3)


def _pages_of(x):
    """Rows ``[n * 64, G, D]`` as pages ``[n, G, 64, D]`` float32."""
    return x.float().view(-1, PAGE, x.shape[1], D).transpose(1, 2)


def _quantised(x):
    """Whole pages ``[n, G, 64, D]`` in 8 bits, and their codes ``[n, G]``."""
    code = _e4m3_code(x.abs().amax((-1, -2)))
    y = x * _power(254 - code)[..., None, None]
    return y.to(torch.float8_e4m3fn), code.to(torch.uint8)


def _lay_out(codes, scales):
    """Weight ``codes [N, K]`` (4-bit E2M1) and ``scales [N, K / 32]`` in the kernel's order.

    Tiles of 16 outputs by 128 inputs: ``[N / 16, K / 128, 64, 16]`` bytes, lane ``16 q + r`` holding
    inputs 32 q to 32 q + 31 of the tile's output r, the even input in a byte's low half.  Scales
    ``[N / 16, K / 512, 64, 4]``: the same lanes, byte i for the i-th of four tiles.  Sizes are
    rounded up, with value 0 and scale 1."""
    n, k = codes.shape
    nt, kc = -(-n // 16), -(-k // 128)
    kc4 = -(-kc // 4)
    full = torch.zeros(nt * 16, kc * 128, dtype=torch.uint8, device=codes.device)
    full[:n, :k] = codes
    packed = full[:, 0::2] | (full[:, 1::2] << 4)
    packed = packed.view(nt, 16, kc, 4, 16).permute(0, 2, 3, 1, 4).reshape(nt, kc, 64, 16)
    s = torch.full((nt * 16, kc4 * 16), 127, dtype=torch.uint8, device=codes.device)
    s[:n, :scales.shape[1]] = scales
    s = s.view(nt, 16, kc4, 4, 4).permute(0, 2, 4, 1, 3).reshape(nt, kc4, 64, 4)
    return packed.contiguous(), s.contiguous()


def _weight_values(packed, scales, n, k):
    """The float32 weight ``[n, k]`` of ``_lay_out``'s tensors."""
    nt, kc = packed.shape[:2]
    kc4 = scales.shape[1]
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=packed.device)
    p = packed.view(nt, kc, 4, 16, 16).permute(0, 3, 1, 2, 4).reshape(nt * 16, kc * 64)
    both = torch.stack((p & 15, p >> 4), -1).view(nt * 16, kc * 4, 32)
    s = scales.view(nt, kc4, 4, 16, 4).permute(0, 3, 1, 4, 2).reshape(nt * 16, kc4 * 16)
    w = table[both.int()] * _power(s[:, :kc * 4])[..., None]
    return w.view(nt * 16, kc * 128)[:n, :k]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _keys_values(rows, G, gen):
    """Keys with a few strong channels and offsets of their own, as after a rotary embedding, and values."""
    gain = torch.exp(0.5 * torch.randn(1, G, D, device=DEV, generator=gen))
    gain[..., :4] *= 6.0
    shift = 0.5 * gain * torch.randn(1, G, D, device=DEV, generator=gen)
    k = torch.randn(rows, G, D, device=DEV, generator=gen) * gain + shift
    v = torch.randn(rows, G, D, device=DEV, generator=gen)
    return k, v


def _cache(batch, longest, G, gen):
    """A cache of ``batch`` sequences; pages past a sequence's end hold what was there before."""
    pages = max(1, -(-longest // PAGE))
    k, v = _keys_values(batch * pages * PAGE, G, gen)
    k8, ks = _quantised(_pages_of(k))
    v8, vs = _quantised(_pages_of(v))
    back = torch.empty_like(v8.view(torch.uint8))
    back[:, :, _place(torch.arange(PAGE, device=DEV))] = v8.view(torch.uint8)
    v8 = back.transpose(2, 3).contiguous().view(torch.float8_e4m3fn)
    shape = (batch, pages, G)
    return dict(k8=k8.contiguous().view(*shape, PAGE, D), v8=v8.view(*shape, D, PAGE),
                k_scale=ks.view(shape).contiguous(), v_scale=vs.view(shape).contiguous())


def _prepare_append(case, gen):
    lens, new, G, dtype = _ints(case["lens"]), _ints(case["new"]), case["G"], DTYPES[case["dtype"]]
    longest = max(a + b for a, b in zip(lens, new))
    st = _cache(len(lens), longest, G, gen)
    kc = torch.randn(len(lens), max(1, _n_windows(st["k8"].shape[1] * PAGE)), G, D, device=DEV,
                     generator=gen)
    k, v = _keys_values(sum(new), G, gen)
    if case["dtype"] == "bf16":  # a strong token now and then raises its page's scale
        k[:: 97] *= 4.0
    return dict(st, kc=kc.to(dtype), k=k.to(dtype), v=v.to(dtype), lens_host=lens,
                cu_host=_cu(new), lens=_i32(lens), cu=_i32(_cu(new)))


def _plan(lens, rows, G, budget, local, gen):
    """Page plans ``[G, batch * rows, take]``: the first page, the row's own and the ``local`` before
    it, and others at random; ascending, then -1."""
    own_page = torch.tensor([(n - rows + i) // PAGE for n in lens for i in range(rows)], device=DEV)
    pages = max(n - 1 for n in lens) // PAGE + 1
    at = torch.arange(pages, device=DEV)
    order = torch.rand(G, len(lens) * rows, pages, device=DEV, generator=gen)
    forced = (at == 0) | ((at <= own_page[:, None]) & (at >= own_page[:, None] - local))
    order = torch.where(forced, order + 1.0, order)
    order = torch.where(at > own_page[:, None], -1.0, order)
    best, ids = order.topk(min(budget, pages), -1)
    ids = torch.where(best < 0, pages, ids).sort(-1).values
    return torch.where(ids == pages, -1, ids).int()


def _prepare_attention(case, gen):
    lens, rows, G, dtype = _ints(case["lens"]), case["rows"], case["G"], DTYPES[case["dtype"]]
    st = _cache(len(lens), max(lens), G, gen)
    q = torch.randn(len(lens) * rows, case["H"], D, device=DEV, generator=gen)
    if case["kind"] == "sparse":
        st["ids"] = _plan(lens, rows, G, case["budget"], case["local"], gen)
    cu = [rows * b for b in range(len(lens) + 1)]
    return dict(st, q=q.to(dtype), lens=_i32(lens), longest=max(lens), rows=rows, cu=_i32(cu),
                causal=case["causal"])


def _prepare_linear(case, gen):
    m, n, k = case["rows"], case["out"], case["inp"]
    w = torch.randn(n, -(-k // 32) * 32, device=DEV, generator=gen) * 0.02
    w[:, k:] = 0.0
    groups = w.view(n, -1, 32)
    scale = _code(groups.abs().amax(-1), 2, 0x400000, 8)  # 6 = 1.5 2^2
    y = groups * _power(254 - scale)[..., None]
    a = y.abs()
    code = sum((a > b).to(torch.uint8) for b in (0.25, 1.25, 2.5, 5.0))
    code += sum((a >= b).to(torch.uint8) for b in (0.75, 1.75, 3.5))
    code |= (y < 0).to(torch.uint8) << 3
    codes, scales = _lay_out(code.view(n, -1)[:, :k], scale.to(torch.uint8))
    x = torch.randn(m, k, device=DEV, generator=gen)
    x[:, :: 251] *= 8.0  # a few strong channels, as after a norm
    return dict(x=x.to(DTYPES[case["dtype"]]), codes=codes, scales=scales, out=n)


_PREPARE = dict(append=_prepare_append, sparse=_prepare_attention, dense=_prepare_attention,
                linear=_prepare_linear, silu=_prepare_linear)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return dict(_PREPARE[case["kind"]](case, gen), kind=case["kind"])


# ---------------------------------------------------------------------------
# One pass: the plain forms
# ---------------------------------------------------------------------------
def _store_plain(x8, scale, new, place, lens, n_new, seq, page, token):
    """Rows ``new [n, G, D]`` into the pages ``x8 [batch, pages, G, 64, D]`` (bytes)."""
    batch, pages, G = scale.shape
    x = new.float()
    slot = seq * pages + page
    top = torch.zeros(batch * pages, G, device=DEV).scatter_reduce_(
        0, slot[:, None].expand(-1, G), x.abs().amax(-1), "amax")
    code = _e4m3_code(top).view(batch, pages, G)
    each = torch.arange(batch, device=DEV)
    begun = (lens // PAGE).clamp(max=pages - 1)
    filled = lens % PAGE
    keeps = ((filled > 0) & (n_new > 0))[:, None]
    before = scale[each, begun].int()
    code[each, begun] = torch.where(keeps, torch.maximum(code[each, begun], before), code[each, begun])
    touched = torch.zeros(batch * pages, dtype=torch.bool, device=DEV)
    touched[slot] = True
    scale.copy_(torch.where(touched.view(batch, pages, 1), code.to(torch.uint8), scale))
    # The rows already in a begun page, under its new scale.
    old = x8[each, begun]
    factor = _power(127 + before - code[each, begun].int().maximum(before))
    again = (old.view(torch.float8_e4m3fn).float() * factor[..., None, None]).to(torch.float8_e4m3fn)
    held = torch.zeros(batch, PAGE, dtype=torch.bool, device=DEV)
    tokens = torch.arange(PAGE, device=DEV)
    held[:, place(tokens)] = tokens < filled[:, None]
    held = (held & keeps)[:, None, :, None]
    x8[each, begun] = torch.where(held, again.view(torch.uint8), old)
    y = x * _power(254 - code.view(-1, G)[slot])[..., None]
    x8[seq, page, :, place(token)] = y.to(torch.float8_e4m3fn).view(torch.uint8)


def _append_plain(st):
    lens, cu = st["lens"].long(), st["cu"].long()
    batch, total = lens.numel(), st["k"].shape[0]
    n_new = cu[1:] - cu[:-1]
    each = torch.arange(batch, device=DEV)
    seq = torch.repeat_interleave(each, n_new, output_size=total)
    pos = lens[seq] + torch.arange(total, device=DEV) - cu[seq]
    where = (lens, n_new, seq, pos // PAGE, pos % PAGE)
    k8 = st["k8"].view(torch.uint8)
    _store_plain(k8, st["k_scale"], st["k"], lambda token: token, *where)
    _store_plain(st["v8"].view(torch.uint8).transpose(-1, -2), st["v_scale"], st["v"], _place, *where)
    # Compressed keys: the mean of 32 stored keys at every 16th token.
    first = torch.where(lens >= 32, (lens - 32) // 16 + 1, 0)
    after = lens + n_new
    count = torch.where(after >= 32, (after - 32) // 16 + 1, 0) - first
    wseq = torch.repeat_interleave(each, count)
    w = first[wseq] + torch.arange(wseq.numel(), device=DEV) - (count.cumsum(0) - count)[wseq]
    p = 16 * w[:, None] + torch.arange(32, device=DEV)
    rows = k8[wseq[:, None], p // PAGE, :, p % PAGE].view(torch.float8_e4m3fn).float()
    rows = rows * _power(st["k_scale"][wseq[:, None], p // PAGE])[..., None]
    st["kc"][wseq, w] = rows.mean(1).to(st["kc"].dtype)


def _attention_plain(st):
    q, G = st["q"], st["k8"].shape[2]
    total, H, _ = q.shape
    lens = st["lens"].long()
    rows = st["rows"]
    seq = torch.arange(total, device=DEV) // rows
    limit = lens[seq] - (rows - 1 - torch.arange(total, device=DEV) % rows if st["causal"] else 0)
    pages = -(-st["longest"] // PAGE)
    if "ids" in st:
        ids = st["ids"].long()
    else:
        ids = torch.arange(pages, device=DEV).expand(G, total, pages)
    at = ids.clamp(min=0)
    group = torch.arange(G, device=DEV)[:, None, None]
    pick = (seq[None, :, None], at, group)
    k = st["k8"].view(torch.uint8)[pick].view(torch.float8_e4m3fn).float()  # [G, rows, take, 64, D]
    k = k * _power(st["k_scale"][pick])[..., None, None]
    v = st["v8"].view(torch.uint8)[pick].view(torch.float8_e4m3fn).float()  # [G, rows, take, D, 64]
    v = v * _power(st["v_scale"][pick])[..., None, None]
    tokens = torch.arange(PAGE, device=DEV)
    v = v[..., _place(tokens)].transpose(-1, -2).reshape(G, total, -1, D)
    k = k.reshape(G, total, -1, D)
    seen = (ids[..., None] >= 0) & (PAGE * at[..., None] + tokens < limit[:, None, None])
    x = q.float().view(total, G, H // G, D).transpose(0, 1)
    s = (x @ k.transpose(-1, -2)) * D ** -0.5
    s = s.masked_fill(~seen.view(G, total, 1, -1), float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.transpose(0, 1).reshape(total, H, D).to(q.dtype)


def _linear_plain(st):
    x = st["x"]
    w = _weight_values(st["codes"], st["scales"], st["out"], x.shape[1])
    y = x.float() @ w.t()
    if st["kind"] == "silu":
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(x.dtype)


def _cache_outputs(st):
    return dict(k=st["k8"], v=st["v8"], k_scale=st["k_scale"], v_scale=st["v_scale"], kc=st["kc"])


def _run_own(st):
    from leanselect_amd import ops

    kind = st["kind"]
    if kind == "append":
        ops.kvcache_append_q8(st["k8"], st["v8"], st["k_scale"], st["v_scale"], st["lens"], st["k"],
                              st["v"], st["cu"], kc_cache=st["kc"], cache_seqlens_host=st["lens_host"],
                              cu_seqlens_new_host=st["cu_host"])
        return _cache_outputs(st)
    if kind == "sparse":
        return ops.sparse_attention_kvcache_q8(
            st["q"], st["k8"], st["v8"], st["k_scale"], st["v_scale"], st["lens"], st["ids"],
            st["cu"], causal=st["causal"])
    if kind == "dense":
        return ops.dense_attention_kvcache_q8(
            st["q"], st["k8"], st["v8"], st["k_scale"], st["v_scale"], st["lens"], st["cu"],
            st["longest"], causal=st["causal"])
    if kind == "linear":
        return ops.linear_mx4(st["x"], st["codes"], st["scales"], st["out"])
    return ops.linear_mx4_silu_mul(st["x"], st["codes"], st["scales"], st["out"])


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "append":
        _append_plain(state)
        return _cache_outputs(state)
    if state["kind"] in ("sparse", "dense"):
        return _attention_plain(state)
    return _linear_plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("linear", "silu"):
        m, n, k = case["rows"], case["out"], case["inp"]
        outputs = n // 2 if kind == "silu" else n
        return {"bytes": n * k / 2 + n * -(-k // 32) + 2.0 * m * k + 2.0 * m * outputs,
                "flops": 2.0 * m * n * k}
    G, lens = case["G"], _ints(case["lens"])
    if kind == "append":
        new = _ints(case["new"])
        windows = [_n_windows(a + b) - _n_windows(a) for a, b in zip(lens, new)]
        old_rows = sum(min(a, 31) for a, w in zip(lens, windows) if w)
        return {"bytes": G * D * (6.0 * sum(new) + old_rows + 2.0 * sum(windows)),
                "flops": G * D * (4.0 * sum(new) + 32.0 * sum(windows))}
    rows, H = case["rows"], case["H"]
    keys = pages = 0.0
    for n in lens:
        have = -(-n // PAGE)
        if kind == "dense":
            keys, pages = keys + rows * n, pages + have
        else:
            take = min(case["budget"], have)
            keys, pages = keys + rows * min(n, take * PAGE), pages + min(have, rows * take)
    return {"bytes": 2.0 * pages * PAGE * G * D + 4.0 * len(lens) * rows * H * D,
            "flops": 4.0 * keys * H * D}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _e4m3_table():
    """The e4m3 magnitudes in order: 0, seven subnormals, then 1.m 2^(e - 7) up to 448."""
    values = [m / 8.0 * 2.0 ** -6 for m in range(8)]
    values += [(1 + m / 8.0) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(values[:-1], dtype=torch.float64, device=DEV)


def _nearest_e4m3(y):
    """The nearest e4m3 value of each, ties to the even one."""
    table = _e4m3_table()
    middle = (table[1:] + table[:-1]) / 2
    a = y.abs()
    low = torch.searchsorted(middle, a)  # a tie goes down
    tie = (low < middle.numel()) & (middle[low.clamp(max=middle.numel() - 1)] == a)
    return torch.copysign(table[low + (tie & (low % 2 == 1)).long()], y)


def _exact_power(e):
    """2^e in float64 for whole e from -254 to 254, from a table: pow rounds on the GPU."""
    table = torch.tensor([2.0 ** i for i in range(-254, 255)], dtype=torch.float64, device=DEV)
    return table[e.long() + 254]


def _least_code(top):
    """The least c >= 1 with top <= 448 2^(c - 127)."""
    return 1 + torch.searchsorted(448.0 * _exact_power(torch.arange(-126, 128, device=DEV)), top)


def _exact_append(case, seed):
    st = prepare(case, seed)
    lens, cu = st["lens_host"], st["cu_host"]
    order = _place(torch.arange(PAGE, device=DEV))
    out = {}
    for name, new in (("k", st["k"].double()), ("v", st["v"].double())):
        # [batch, pages, 64 tokens, G, D], by token
        x = st[name + "8"].double()
        x = (x.permute(0, 1, 3, 2, 4) if name == "k" else x[..., order].permute(0, 1, 4, 2, 3)).contiguous()
        codes = st[name + "_scale"].long()
        for b, before in enumerate(lens):
            rows = new[cu[b]:cu[b + 1]]
            if not len(rows):
                continue
            begin, end = before // PAGE, -(-(before + len(rows)) // PAGE)
            lead, tail = before - begin * PAGE, end * PAGE - before - len(rows)
            nothing = torch.zeros(1, *rows.shape[1:], dtype=torch.float64, device=DEV)
            padded = torch.cat((nothing.expand(lead, -1, -1), rows, nothing.expand(tail, -1, -1)))
            padded = padded.view(end - begin, PAGE, *rows.shape[1:])
            code = _least_code(padded.abs().amax((1, 3)))
            part = x[b, begin:end]
            if lead:
                code[0] = torch.maximum(code[0], codes[b, begin])
                shrink = _exact_power(codes[b, begin] - code[0])
                part[0, :lead] = _nearest_e4m3(part[0, :lead] * shrink[:, None])
            put = _nearest_e4m3(padded * _exact_power(127 - code)[:, None, :, None])
            flat = part.view(-1, *rows.shape[1:])
            flat[lead:lead + len(rows)] = put.view(flat.shape)[lead:lead + len(rows)]
            codes[b, begin:end] = code
        out[name + "_scale"] = codes.to(torch.uint8)
        out[name] = x
    kc = st["kc"].double()
    held = out["k"] * _exact_power(out["k_scale"].long() - 127)[:, :, None, :, None]
    for b, before in enumerate(lens):
        flat = held[b].reshape(-1, *held.shape[3:])
        for w in range(_n_windows(before), _n_windows(before + cu[b + 1] - cu[b])):
            kc[b, w] = flat[16 * w:16 * w + 32].mean(0)
    v = torch.empty_like(out["v"])
    v[:, :, order] = out["v"]
    return dict(k=out["k"].permute(0, 1, 3, 2, 4).contiguous(), v=v.permute(0, 1, 3, 4, 2).contiguous(),
                k_scale=out["k_scale"], v_scale=out["v_scale"], kc=kc)


def _exact_attention(case, seed):
    st = prepare(case, seed)
    q = st["q"].double()
    total, H, _ = q.shape
    G, rows = case["G"], case["rows"]
    order = _place(torch.arange(PAGE, device=DEV))
    out = torch.zeros_like(q)
    for t in range(total):
        b, i = divmod(t, rows)
        n = _ints(case["lens"])[b]
        limit = n - (rows - 1 - i) if case["causal"] else n
        for g in range(G):
            pages = torch.arange(-(-n // PAGE), device=DEV)
            if case["kind"] == "sparse":
                plan = st["ids"][g, t].long()
                pages = plan[plan >= 0]
            k = st["k8"].view(torch.uint8)[b, pages, g].view(torch.float8_e4m3fn).double()
            v = st["v8"].view(torch.uint8)[b, pages, g].view(torch.float8_e4m3fn).double()
            k = k * _exact_power(st["k_scale"][b, pages, g].long() - 127)[:, None, None]
            v = v * _exact_power(st["v_scale"][b, pages, g].long() - 127)[:, None, None]
            pos = (PAGE * pages[:, None] + torch.arange(PAGE, device=DEV)).view(-1)
            seen = pos < limit
            k = k.reshape(-1, D)[seen]
            v = v[..., order].transpose(1, 2).reshape(-1, D)[seen]
            heads = slice(g * H // G, (g + 1) * H // G)
            out[t, heads] = torch.softmax(q[t, heads] @ k.t() / math.sqrt(D), -1) @ v
    return out


def _exact_linear(case, seed):
    st = prepare(case, seed)
    n, k = case["out"], case["inp"]
    x = st["x"].double()
    codes, scales = st["codes"], st["scales"]
    y = torch.empty(x.shape[0], codes.shape[0] * 16, dtype=torch.float64, device=DEV)
    magnitude = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    x = torch.nn.functional.pad(x, (0, codes.shape[1] * 128 - k))
    for at in range(0, codes.shape[0], 256):
        c = codes[at:at + 256].long()
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2)  # [tiles, chunks, lane, 32]
        w = magnitude[c & 7] * (1 - 2 * (c >> 3))
        s = scales[at:at + 256].permute(0, 1, 3, 2).flatten(1, 2)[:, :c.shape[1]]
        w = w * _exact_power(s.long() - 127)[..., None]
        w = w.view(*w.shape[:2], 4, 16, 32).permute(0, 3, 1, 2, 4).reshape(w.shape[0] * 16, -1)
        y[:, at * 16:at * 16 + w.shape[0]] = x @ w.t()
    y = y[:, :n]
    if case["kind"] == "silu":
        y = y[:, :n // 2] * torch.sigmoid(y[:, :n // 2]) * y[:, n // 2:]
    return y.contiguous()


def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    return (_exact_linear if case["kind"] in ("linear", "silu") else _exact_attention)(case, seed)
