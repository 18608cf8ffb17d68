"""Patched encoder modules beside the modules they replace: calls in which the two must not differ in what they compute."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ea():
    from morphik_core_amd import encoder_attention

    assert torch.cuda.is_available()
    yield encoder_attention
    torch.cuda.empty_cache()


def gemma(**config):
    """A small random Gemma decoder in bf16 on the GPU."""
    from transformers import GemmaConfig, GemmaModel

    cfg = GemmaConfig(**{**dict(hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=32, vocab_size=100), **config})
    torch.manual_seed(3)
    return GemmaModel(cfg).to(torch.bfloat16).cuda().eval()


def ids(batch=2, rows=9, seed=4):
    return torch.randint(1, 100, (batch, rows), generator=torch.Generator().manual_seed(seed)).cuda()


def near(a, b):
    """Hidden states of unit scale after two bf16 blocks: sums of roundings of 2^-8 each, far below what one wrong key does to a row."""
    off = (a.float() - b.float()).norm(dim=-1) / b.float().norm(dim=-1)
    return float(off.max()) < 0.05


def test_a_prompt_in_front_of_an_empty_static_cache_sees_itself_only(ea):
    """The cache hands back all of its places, the mask is left to `causal`: row i sees the keys up to i, not the unfilled ones behind them."""
    from transformers import StaticCache

    model, x = gemma(), ids()
    with torch.inference_mode():
        plain = model(input_ids=x).last_hidden_state
        ea.patch_attention(model)
        want = model(input_ids=x).last_hidden_state
        cache = StaticCache(config=model.config, max_cache_len=40)
        got = model(input_ids=x, past_key_values=cache, use_cache=True).last_hidden_state
        assert torch.equal(got, want) and near(want, plain)
        nxt = ids(rows=1, seed=5)  # and the token behind it, whose mask is one of key ranges
        got = model(input_ids=nxt, past_key_values=cache, use_cache=True).last_hidden_state
        assert near(got, model(input_ids=torch.cat([x, nxt], 1)).last_hidden_state[:, -1:])


def test_without_a_mask_the_forward_then_the_module_say_whether_rows_are_causal(ea):
    """is_causal= of a forward reaches the blocks; a module that says nothing counts as causal, as for the framework's own function."""
    from transformers import AttentionInterface

    model, x = gemma(), ids()
    with torch.inference_mode():
        plain = [model(input_ids=x, **kw).last_hidden_state for kw in ({}, dict(is_causal=False), dict(is_causal=True))]
        assert not near(plain[0], plain[1])
        ea.patch_attention(model)
        for want, kw in zip(plain, ({}, dict(is_causal=False), dict(is_causal=True))):
            assert near(model(input_ids=x, **kw).last_hidden_state, want)

    class Says(torch.nn.Module):
        def __init__(self, **said):
            super().__init__()
            for name, value in said.items():
                setattr(self, name, value)

    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(1, 2, 7, 32, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    with torch.inference_mode():
        for module in (Says(), Says(is_causal=True), Says(is_causal=False)):
            for asked in (None, True, False):
                got = ea._interface_attention(module, q, k, v, is_causal=asked)[0]
                assert near(got, AttentionInterface()["sdpa"](module, q, k, v, None, is_causal=asked)[0])


def test_dropout_of_a_model_in_training_mode_stays(ea):
    """Under no_grad too: the same bits as the unpatched model from the same random state; in evaluation mode the kernels run again."""
    x = ids()
    padded = torch.ones_like(x)
    padded[1, 5:] = 0
    model = gemma(attention_dropout=0.5).train()

    def run(seed, mask):
        torch.manual_seed(seed)
        with torch.no_grad():
            return model(input_ids=x, attention_mask=mask).last_hidden_state

    plain = [run(s, m) for s in (1, 2) for m in (None, padded)]
    ea.patch_attention(model)
    got = [run(s, m) for s in (1, 2) for m in (None, padded)]
    assert torch.equal(got[0], plain[0]) and torch.equal(got[2], plain[2]) and not near(got[0], got[2])
    assert all(near(a[padded.bool()], b[padded.bool()]) for a, b in zip(got, plain))
    model.eval()
    assert not near(run(1, None), plain[0]) and torch.equal(run(1, None), run(2, None))


@pytest.mark.parametrize("how", ["module", "global", "wrapped"])
def test_what_a_projection_returned_stays_as_it_was(ea, how):
    """A forward hook that keeps the outputs of q_proj and k_proj sees the projections, not their rotated values; so does a layer that keeps its own output."""
    kept = {}

    def keep(module, args, out):
        if isinstance(module, torch.nn.Linear):
            kept[module] = (args[0], out)

    class Keeping(torch.nn.Linear):
        def forward(self, x):
            out = super().forward(x)
            keep(self, (x,), out)
            return out

    model, x = gemma(), ids()
    with torch.inference_mode():
        ea.patch_attention(model)
        want = model(input_ids=x).last_hidden_state
        blocks = [layer.self_attn for layer in model.layers]
        handles = []
        if how == "module":
            handles = [p.register_forward_hook(keep) for b in blocks for p in (b.q_proj, b.k_proj)]
        elif how == "global":
            handles = [torch.nn.modules.module.register_module_forward_hook(keep)]
        else:
            for b in blocks:
                for p in (b.q_proj, b.k_proj):
                    p.__class__ = Keeping
        try:
            assert torch.equal(model(input_ids=x).last_hidden_state, want)
        finally:
            for h in handles:
                h.remove()
        for b in blocks:
            for p in (b.q_proj, b.k_proj):
                seen, out = kept[p]
                assert torch.equal(out, torch.nn.functional.linear(seen, p.weight, p.bias))


def test_frequencies_that_change_after_the_first_forward_are_used(ea):
    """Assigned anew, changed in place, cast with the model, another attention_scaling: each forward turns by what the rotary module holds then."""
    model, plain, x = gemma(), gemma(), ids(rows=60)
    for m in (model, plain):
        for layer in m.layers:  # scores of about 1: of the random weights as they are every row is nearly the mean of its keys, however it is turned
            layer.self_attn.q_proj.weight.data *= 5
            layer.self_attn.k_proj.weight.data *= 5
    ea.patch_attention(model)

    def assign(m):
        m.rotary_emb.inv_freq = m.rotary_emb.inv_freq * 3

    def in_place(m):
        m.rotary_emb.inv_freq.mul_(0.2)

    def scaling(m):
        m.rotary_emb.attention_scaling = 0.5

    def cast(m):
        m.to(torch.float16)

    with torch.inference_mode():
        last = model(input_ids=x).last_hidden_state
        for change in (assign, scaling):
            change(model), change(plain)
            got, want = model(input_ids=x).last_hidden_state, plain(input_ids=x).last_hidden_state
            assert near(got, want) and not near(got, last), change.__name__
            last = got
    for change in (in_place, cast):
        with torch.no_grad():
            model.rotary_emb.inv_freq, plain.rotary_emb.inv_freq = (torch.arange(16, 0, -1, device="cuda") / 7.0 for _ in range(2))
            model(input_ids=x)
            change(model), change(plain)
            got, want = model(input_ids=x).last_hidden_state, plain(input_ids=x).last_hidden_state
            assert near(got, want), change.__name__
    table = model.rotary_emb._mv_rotary_table
    with torch.no_grad():
        model(input_ids=x)
    assert model.rotary_emb._mv_rotary_table is table  # and not made again where nothing changed


def test_calls_that_the_kernel_does_not_take_fall_back(ea):
    """Values of another width than the keys, rows of K further apart than the kernel reaches, a cache that hands back another layout: the framework's function
    answers, where `attention` itself refuses."""
    from transformers import AttentionInterface, DynamicCache

    class Module(torch.nn.Module):
        is_causal = False

    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(1, h, n, d, generator=g, device="cuda").to(torch.bfloat16) for h, n, d in ((2, 5, 32), (2, 3, 32), (2, 3, 16)))
    far = torch.zeros(2 * (1 << 23) + 4096, dtype=torch.bfloat16, device="cuda").as_strided((1, 2, 2, 32), (64, 32, (1 << 23) + 8, 1))
    far.copy_(k[:, :, :2])
    with torch.inference_mode():
        for args in ((q, k, v), (q, far, far), (q, far, k[:, :, :2])):
            got = ea._interface_attention(Module(), *args)[0]
            assert near(got, AttentionInterface()["sdpa"](Module(), *args, None)[0])

        class Odd(DynamicCache):
            def update(self, *args, **kwargs):
                return tuple(torch.nn.functional.pad(t, (0, 4))[..., :-4] for t in super().update(*args, **kwargs))

        model, x = gemma(), ids()
        want = model(input_ids=x).last_hidden_state
        ea.patch_attention(model)
        assert near(model(input_ids=x, past_key_values=Odd(config=model.config), use_cache=True).last_hidden_state, want)


def test_a_patched_decoder_captured_into_a_graph_follows_its_inputs(ea):
    """Captured once, replayed with new embeddings copied in and eager forwards between the replays.  While capturing the framework hands over a mask, and whether it
    is one of ranges cannot be asked then: the graph holds the modules' own attention, so it is near the eager forward and the unpatched one, not bit-equal."""
    model, plain = gemma(), gemma()
    ea.patch_attention(model)
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(2, 33, 128, generator=g, device="cuda").to(torch.bfloat16)

    def body(m=model):
        return m(inputs_embeds=x, use_cache=False).last_hidden_state

    with torch.inference_mode():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = body()
        for _ in range(4):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            eager, want = body(), body(plain)
            got = []
            for _ in range(2):
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                got.append(out.clone())
            assert torch.equal(*got) and near(got[0], want) and near(eager, want)
