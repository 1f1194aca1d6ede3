"""The recurrent decode engine over the 8-bit cache and with sampled tokens, and the serving layer's options for both."""
import pytest
import torch

from recurrent_pretraining_b200.config import ModelConfig

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from recurrent_pretraining_b200.models.hf import RavenForCausalLM

    torch.manual_seed(0)
    cfg = ModelConfig.from_name("smoke-raven-96", mean_recurrence=4)
    return RavenForCausalLM.from_training_model(cfg.construct_model()).to(torch.bfloat16).cuda().eval()


def nearly_largest(model, toks, P):
    """Whether the tokens behind the first P are (nearly) the largest logits of the eager model on these tokens.  The products of a decode step
    add their parts atomically, so two runs differ in last bits, now and then in a code of the cache, and at a tie in a token: runs are held
    against the model, not against each other."""
    pred = model(toks[:, :-1], num_steps=4, init_scale=0.0).logits[:, P - 1:, :].float()
    chosen = torch.gather(pred, -1, toks[:, P:].unsqueeze(-1)).squeeze(-1)
    return bool((chosen >= pred.max(-1).values - 0.15 - 0.25 * pred.std(-1)).all())


@gpu
@pytest.mark.parametrize("use_graphs,B,P,strategy", [(False, 2, 24, "full"), (True, 3, 41, "full"), (True, 2, 33, "full-compress-s4")])
def test_engine_over_the_8bit_cache(model, use_graphs, B, P, strategy):
    """The engine's tokens are (nearly) the largest logits of a cache whose values were rounded to e4m3: the eager model on the engine's
    own tokens differs by that rounding, whose effect on these logits is far below their spread."""
    from recurrent_pretraining_b200.engine.decode import DecodeEngine

    torch.manual_seed(1)
    new = 9
    ids = torch.randint(0, 4000, (B, P), device="cuda")
    eng = DecodeEngine(model, max_batch=B, max_len=61, num_steps=4, use_graphs=use_graphs, cache_lookup_strategy=strategy, kv_dtype="fp8")
    toks, stats = eng.generate(ids, new, init_scale=0.0)
    assert stats["device_status"] == 0 and toks.shape == (B, P + new)
    again, _ = eng.generate(ids, new, init_scale=0.0)      # reused rows need no clearing
    if "compress" not in strategy:
        assert nearly_largest(model, toks, P) and nearly_largest(model, again, P)
    half = DecodeEngine(model, max_batch=B, max_len=61, num_steps=4, cache_lookup_strategy=strategy)
    assert eng.cache.get_memory_usage() < 0.56 * half.cache.get_memory_usage()


@gpu
def test_graphs_over_the_8bit_cache_change_nothing(model):
    from recurrent_pretraining_b200.engine.decode import DecodeEngine

    ids = torch.randint(0, 4000, (3, 30), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    outs = [DecodeEngine(model, 3, 64, num_steps=4, use_graphs=g, kv_dtype="fp8").generate(ids, 12, init_scale=0.0)[0] for g in (False, True)]
    assert all(nearly_largest(model, o, 30) for o in outs)


@gpu
def test_kl_exit_and_programmatic_launch_over_the_8bit_cache(model, monkeypatch):
    from recurrent_pretraining_b200.engine import decode as D

    torch.manual_seed(2)
    ids = torch.randint(0, 4000, (2, 16), device="cuda")
    eng = D.DecodeEngine(model, max_batch=2, max_len=48, num_steps=4, max_steps=8, kv_dtype="fp8")
    toks, reuse = eng.generate(ids, 4, criterion="kl", exit_threshold=5e-4, max_steps=8, continuous_compute=True)
    assert toks.shape == (2, 20) and reuse["device_status"] == 0
    plain, _ = eng.generate(ids, 8, init_scale=0.0)
    monkeypatch.setattr(D, "PDL", True)
    toks, stats = D.DecodeEngine(model, max_batch=2, max_len=48, num_steps=4, max_steps=8, kv_dtype="fp8").generate(ids, 8, init_scale=0.0)
    assert stats["device_status"] == 0 and nearly_largest(model, toks, 16) and nearly_largest(model, plain, 16)


@gpu
def test_a_prompt_in_two_chunks_reads_the_decoded_cache(model):
    from recurrent_pretraining_b200.engine.decode import StaticRecurrentKV8Cache

    cache = StaticRecurrentKV8Cache(3, 2, 50, 5, 96, "cuda", 2, 4, 2)
    k = torch.randn(2, 40, 5, 96, device="cuda").to(torch.bfloat16)
    a, _ = cache.update(k[:, :25], k[:, :25], 0)
    assert a.data_ptr() == k.data_ptr()
    b, c = cache.update(k[:, 25:], -k[:, 25:], 0)
    assert b.shape == (2, 40, 5, 96)
    assert ((b.float() - k.float()).abs() <= 2.0 ** -4 * k.float().abs() + 2.0 ** -9).all()     # one rounding to e4m3, or two where a block grew
    assert ((c[:, 25:].float() + k[:, 25:].float()).abs() <= 2.0 ** -4 * k[:, 25:].float().abs() + 2.0 ** -9).all()


@gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_sampled_tokens(model, kv_dtype):
    """Sampling is what ``sample_tokens`` draws from the engine's own logits with the generator's numbers, and the narrowest filters are
    greedy."""
    from recurrent_pretraining_b200.engine.decode import DecodeEngine
    from recurrent_pretraining_b200.models.sampling import SamplingOptions
    from recurrent_pretraining_b200.ops.sampling import sample_tokens

    ids = torch.randint(0, 4000, (2, 20), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    eng = DecodeEngine(model, max_batch=2, max_len=64, num_steps=4, kv_dtype=kv_dtype)
    run = lambda seed, **o: eng.generate(ids, 10, init_scale=0.0, sampling=SamplingOptions(do_sample=True, **o),  # noqa: E731
                                         generator=torch.Generator("cuda").manual_seed(seed))[0]
    assert all(nearly_largest(model, run(1, **narrow), 20) for narrow in (dict(top_k=1), dict(top_p=1e-9), dict(min_p=1.0)))
    assert not torch.equal(run(7, temperature=1.5, top_k=200, top_p=0.95), run(8, temperature=1.5, top_k=200, top_p=0.95))
    logits = torch.randn(2, 4096, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    numbers = torch.rand(2, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    options = dict(temperature=1.5, top_k=200, top_p=0.95)
    eng.uniform[:2] = numbers
    assert torch.equal(eng._pick(logits, eng._settings(SamplingOptions(do_sample=True, **options))), sample_tokens(logits, numbers, **options))
    graphs = len(eng._graphs)
    for t in (0.3, 0.31, 0.32):
        run(9, temperature=t, top_p=0.5 + t)
    assert len(eng._graphs) == graphs                        # requests' settings need no graphs of their own
    for bad in (dict(temperature=-1.0), dict(top_k=-2), dict(top_p=1.5), dict(min_p=-0.1)):
        with pytest.raises(ValueError):
            run(9, **bad)
    assert nearly_largest(model, eng.generate(ids, 10, init_scale=0.0, sampling=SamplingOptions(temperature=3.0))[0], 20)      # do_sample is off
    with pytest.raises(ValueError):
        eng.generate(ids, 4, criterion="kl", sampling=SamplingOptions(do_sample=True))
    with pytest.raises(ValueError):
        eng.generate(ids, 4, sampling=SamplingOptions(do_sample=True, repetition_penalty=1.2))


@gpu
def test_served_with_sampling_over_the_8bit_cache(model):
    from recurrent_pretraining_b200.engine import server as S

    sched = S.BatchScheduler(S.make_backend(model, max_batch=2, max_len=64, kv_dtype="fp8"), window_ms=20.0, stop_ids=())
    try:
        body = {"prompt": [5, 17, 3], "max_tokens": 6, "num_steps": 4, "init_scale": 0.0}
        for options in ({}, {"do_sample": True, "top_k": 1}):
            tokens = S.handle_completion(sched, {**body, **options})["choices"][0]["token_ids"]
            assert nearly_largest(model, torch.tensor([body["prompt"] + tokens], device="cuda"), 3)
        assert len(S.handle_completion(sched, {**body, "do_sample": True, "temperature": 0.8, "top_p": 0.9})["choices"][0]["token_ids"]) == 6
        with pytest.raises(RuntimeError):
            S.handle_completion(sched, {**body, "do_sample": True, "criterion": "kl"})
    finally:
        sched.close()


def test_an_8bit_cache_is_refused_where_there_is_none():
    from recurrent_pretraining_b200.engine import server as S

    class Tiny(torch.nn.Linear):
        pass

    with pytest.raises(ValueError):
        S.make_backend(Tiny(2, 2), kv_dtype="fp8")


# Weights of a temperature this high are equal whatever the logits are, so the token is the number's place in the vocabulary: floor(u V).
FLAT = dict(do_sample=True, temperature=1e30)


def places(generator, B, V, steps):
    return torch.stack([(torch.empty(B, device="cuda").uniform_(generator=generator).double() * V).floor().long() for _ in range(steps)], 1)


@gpu
def test_prefill_draws_from_numbers_of_its_own(model):
    from recurrent_pretraining_b200.engine.decode import DecodeEngine
    from recurrent_pretraining_b200.models.sampling import SamplingOptions

    ids = torch.randint(0, 4000, (2, 20), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    eng = DecodeEngine(model, max_batch=2, max_len=64, num_steps=4)
    flat = SamplingOptions(**FLAT)
    first, second = (eng.prefill(ids, init_scale=0.0, sampling=flat) for _ in range(2))
    assert not torch.equal(first, second)
    drawn = eng.prefill(ids, init_scale=0.0, sampling=flat, generator=torch.Generator("cuda").manual_seed(3))
    assert torch.equal(drawn, places(torch.Generator("cuda").manual_seed(3), 2, eng.V, 1)[:, 0])


def test_a_request_with_a_temperature_of_zero_is_greedy():
    from recurrent_pretraining_b200.engine import server as S

    cold, none = S.DecodeOptions(do_sample=True, temperature=0.0), S.DecodeOptions(do_sample=True)
    assert cold.sampling() == {} and none.sampling() == {"do_sample": True}
    assert cold.key() != none.key() and cold.key() == S.DecodeOptions().key()
    off = S.DecodeOptions(do_sample=True, temperature=0.7, top_k=0, top_p=0.0, min_p=0.0)                  # filters of zero are off, as if not given
    assert off.sampling() == {"do_sample": True, "temperature": 0.7}


@gpu
def test_a_temperature_of_zero_takes_the_largest_logit(model):
    """As ``sample_tokens`` does: not a draw at another temperature."""
    from recurrent_pretraining_b200.engine import server as S
    from recurrent_pretraining_b200.engine.decode import DecodeEngine
    from recurrent_pretraining_b200.models.sampling import SamplingOptions

    ids = torch.randint(0, 4000, (2, 20), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    eng = DecodeEngine(model, max_batch=2, max_len=64, num_steps=4)
    cold = SamplingOptions(do_sample=True, temperature=0.0)
    logits = torch.randn(2, 4096, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    logits[1, [7, 4000]] = 9.0
    eng.uniform.fill_(0.75)
    assert torch.equal(eng._pick(logits, eng._settings(cold)), torch.stack([logits[0].argmax(), torch.tensor(7, device="cuda")]))
    assert nearly_largest(model, eng.generate(ids, 10, init_scale=0.0, sampling=cold)[0], 20)
    sched = S.BatchScheduler(S.make_backend(model, max_batch=2, max_len=64), window_ms=5.0, stop_ids=())
    try:
        body = {"prompt": [5, 17, 3], "max_tokens": 8, "num_steps": 4, "init_scale": 0.0, "do_sample": True, "temperature": 0}
        tokens = S.handle_completion(sched, body)["choices"][0]["token_ids"]
        assert nearly_largest(model, torch.tensor([body["prompt"] + tokens], device="cuda"), 3)
    finally:
        sched.close()


@gpu
@pytest.mark.parametrize("new", [1, 3])
def test_rows_without_a_finite_logit_are_reported(model, new):
    """Also where the token is the last one of a request, which no later step looks up."""
    from recurrent_pretraining_b200.engine import server as S
    from recurrent_pretraining_b200.engine.decode import DecodeEngine
    from recurrent_pretraining_b200.models.sampling import SamplingOptions

    ids = torch.randint(0, 4000, (2, 12), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    hot = SamplingOptions(do_sample=True, temperature=1.0)
    eng = DecodeEngine(model, max_batch=2, max_len=32, num_steps=4)
    keep = model.lm_head.weight.detach().clone()
    try:
        with torch.no_grad():
            model.lm_head.weight.fill_(float("nan"))
        _, stats = eng.generate(ids, new, init_scale=0.0, sampling=hot)
        assert stats["device_status"] != 0
        backend = S.make_backend(model, max_batch=1, max_len=32)
        with pytest.raises(RuntimeError):
            backend.generate([[5, 17, 3]], S.DecodeOptions(max_tokens=new, num_steps=4, init_scale=0.0, do_sample=True))
    finally:
        with torch.no_grad():
            model.lm_head.weight.copy_(keep)
    tokens, stats = eng.generate(ids, new, init_scale=0.0, sampling=hot)
    assert stats["device_status"] == 0 and (tokens >= 0).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_second_chunk_decodes_what_it_reads(device):
    """The codes of the positions so far, not of the capacity."""
    from recurrent_pretraining_b200.engine.decode import StaticRecurrentKV8Cache

    cache = StaticRecurrentKV8Cache(1, 2, 5000, 5, 96, device, 1, 0, 0)
    k = torch.randn(2, 70, 5, 96, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(device)
    cache.update(k[:, :33], k[:, :33], 0)
    for got in cache.update(k[:, 33:], k[:, 33:], 0):
        assert got.shape == (2, 70, 5, 96) and got.untyped_storage().nbytes() == k.untyped_storage().nbytes()
        assert ((got.float() - k.float()).abs() <= 2.0 ** -3 * k.float().abs() + 2.0 ** -8).all()          # two roundings to e4m3 at most


@gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("use_graphs", [False, True])
def test_every_sampled_token_is_drawn_from_the_generators_numbers(model, use_graphs, kv_dtype):
    from recurrent_pretraining_b200.engine.decode import DecodeEngine
    from recurrent_pretraining_b200.models.sampling import SamplingOptions

    ids = torch.randint(0, 4000, (3, 20), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    eng = DecodeEngine(model, max_batch=3, max_len=64, num_steps=4, use_graphs=use_graphs, kv_dtype=kv_dtype)
    for seed in (3, 4):
        toks, _ = eng.generate(ids, 12, init_scale=0.0, sampling=SamplingOptions(**FLAT), generator=torch.Generator("cuda").manual_seed(seed))
        assert torch.equal(toks[:, 20:], places(torch.Generator("cuda").manual_seed(seed), 3, eng.V, 12))


def test_numbers_take_their_place_where_weights_are_equal():
    from recurrent_pretraining_b200.ops.sampling import sample_tokens

    u = torch.rand(500, generator=torch.Generator().manual_seed(1))
    x = torch.randn(500, 4096, generator=torch.Generator().manual_seed(2))
    assert torch.equal(sample_tokens(x, u, temperature=1e30), (u.double() * 4096).floor().long())


@gpu
@pytest.mark.parametrize("strategy", ["full", "full-compress-s4", "full-compress-s1"])
def test_slots_of_the_8bit_cache_hold_what_the_bf16_cache_holds(model, strategy):
    """Both engines over the same tokens.  A prompt's slots differ by one rounding to e4m3 of equal values; those of later tokens, whose hidden states saw
    rounded keys and values (3 % of noise each), by far less than a wrong exponent (a factor of two) would make of them."""
    from recurrent_pretraining_b200.engine.decode import DecodeEngine

    B, P, steps = 2, 41, 9
    ids = torch.randint(0, 4000, (B, P + steps), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    half, fp8 = (DecodeEngine(model, max_batch=B, max_len=64, num_steps=4, cache_lookup_strategy=strategy, kv_dtype=t) for t in ("bf16", "fp8"))

    def slots():
        for s in range(half.cache.n_slots):
            yield from zip((half.cache.k[s].float(), half.cache.v[s].float()), (t[:, :half.Lmax].float() for t in fp8.cache.layers[s].decoded()),
                           (fp8.cache.k_exp[s], fp8.cache.v_exp[s]))

    with torch.no_grad():
        for eng in (half, fp8):
            eng.prefill(ids[:, :P], init_scale=0.0)
        for want, got, exps in slots():
            step = torch.exp2(exps.float()).repeat_interleave(32, -1)[:, :, :half.Lmax].transpose(1, 2)[..., None]         # of a code below 2^-6
            tol = (2.0 ** -4 + 2.0 ** -8) * want.abs() + 2.0 ** -10 * step
            assert ((got - want).abs() <= tol)[:, :P].all()
        for i in range(steps):
            logits = []
            for eng in (half, fp8):
                eng.tok.copy_(ids[:, P + i])
                eng._fresh_state(0.0)
                eng._token_fixed(4, False)
                eng.pos.add_(1)
                eng.lens.add_(1)
                logits.append(eng.logits.float())
            assert ((logits[0] - logits[1]).abs() <= 0.15 + 0.25 * logits[0].std(-1, keepdim=True)).all()
        for want, got, _ in slots():
            for at in range(P, P + steps):
                assert (got[:, at] - want[:, at]).norm() <= 0.15 * want[:, at].norm()
            assert (got[:, :P] - want[:, :P]).norm() <= 0.15 * want[:, :P].norm()


@gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_kl_decoding_that_never_exits_is_greedy_decoding(model, kv_dtype):
    """A threshold that no divergence is below: every token takes all recurrences and is (nearly) the model's largest logit."""
    from recurrent_pretraining_b200.engine.decode import DecodeEngine

    ids = torch.randint(0, 4000, (2, 16), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    eng = DecodeEngine(model, max_batch=2, max_len=48, num_steps=4, kv_dtype=kv_dtype)
    toks, stats = eng.generate(ids, 9, criterion="kl", exit_threshold=-1.0, max_steps=4, init_scale=0.0)
    assert stats["device_status"] == 0 and stats["steps"] == [[4, 4]] * 8
    assert nearly_largest(model, toks, 16)
