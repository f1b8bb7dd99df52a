"""The model's decode step over the 8-bit cache: its attention is that of its cache."""
import pytest
import torch

from leanselect_amd import minicpm
from oracle import lowbit_oracle as lo
from test_gpu_decode_q8 import DEV, _check

pytestmark = pytest.mark.gpu


def _model(dtype):
    cfg = minicpm.MiniCPMConfig(hidden_size=1024, num_hidden_layers=2, num_attention_heads=8,
                                num_key_value_heads=2, intermediate_size=2048, vocab_size=4096,
                                topk=8, local_blocks=4)
    return minicpm.MiniCPMLeanSelect(cfg, device=DEV, dtype=dtype, seed=7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_step_attends_its_own_cache(dtype):
    """Each layer of each step: the new rows are the ones appended (byte for byte what the
    definition makes of the cache before), and what goes on is their 64-bit attention, over the
    layer's own pages and plan.  The same step with that attention in place of the kernel's gives
    the same logits up to roundings; with the first layer's in both, or none, it does not."""
    model = _model(dtype)
    g = torch.Generator(device=DEV).manual_seed(13)
    ids = torch.randint(0, 4096, (1200,), generator=g, device=DEV, dtype=torch.int32)
    caches = {}
    for name in ("kernel", "oracle", "first layer", "nothing"):
        caches[name] = model.new_cache(2, 1024, kv_format="q8")
        model.prefill(ids, [0, 300, 1200], cache=caches[name])
    steps = []

    def watch(cache):
        before = [lo.Q8Cache(*cache.layer(i)) for i in range(2)]
        update, attend = cache.update, cache.attend

        def updated(layer, k, v):
            before[layer].append(cache.lengths, k.cpu(), v.cpu(), [0, 1, 2])
            update(layer, k, v)
            got, want = lo.Q8Cache(*cache.layer(layer)), before[layer]
            for b, n in enumerate(cache.lengths_after):
                page, row = (n - 1) // 64, (n - 1) % 64
                for a, c in ((got.k, want.k), (got.v, want.v)):
                    assert torch.equal(a[b, page, :, :row + 1], c[b, page, :, :row + 1])
                for a, c in ((got.kcode, want.kcode), (got.vcode, want.vcode)):
                    assert torch.equal(a[b, :page + 1], c[b, :page + 1])

        def attended(layer, q, plan, cu, **kw):
            out = attend(layer, q, plan, cu, **kw)
            want, _, bound = lo.attend(lo.Q8Cache(*cache.layer(layer)), q.cpu(), cache.lengths_after,
                                       [0, 1, 2], plan.cpu())
            _check(out, None, want, None, bound, dtype)
            steps.append(layer)
            return out

        cache.update, cache.attend = updated, attended

    def oracle(cache, first):
        def attended(layer, q, plan, cu, **kw):
            of = 0 if first else layer
            want, _, _ = lo.attend(lo.Q8Cache(*cache.layer(of)), q.cpu(), cache.lengths_after, [0, 1, 2],
                                   plan.cpu())
            return want.to(dtype).to(DEV)

        cache.attend = attended

    watch(caches["kernel"])
    oracle(caches["oracle"], False)
    oracle(caches["first layer"], True)
    caches["nothing"].attend = lambda layer, q, *a, **kw: torch.zeros_like(q)
    for _ in range(3):
        tok = torch.randint(0, 4096, (2,), generator=g, device=DEV, dtype=torch.int32)
        logits = {name: model.decode_step(tok, cache) for name, cache in caches.items()}
        off = {name: ((x - logits["kernel"]).norm() / logits["kernel"].norm()).item()
               for name, x in logits.items()}
        # Attention in the kernel and in 64 bits, each rounded once: a step of the type apart in
        # few places; then two layers of some ten roundings each.  (Measured: the same bits;
        # without attention 0.2.)
        eps = torch.finfo(dtype).eps / 2
        assert off["oracle"] <= 20 * eps, off
        assert min(off["first layer"], off["nothing"]) > 20 * eps, off
    assert steps == [0, 1] * 3
