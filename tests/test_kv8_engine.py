"""The engine over an 8-bit KV cache, and with controls of logits."""
import json

import pytest
import torch

from k8s_llm_monitor_amd.engine import EngineConfig, LLMEngine, SamplingParams
from k8s_llm_monitor_amd.engine.engine import EngineService

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GREEDY = dict(temperature=0.0, ignore_eos=True)


def engine(dev, **kw):
    kw = {"model": "llama-tiny-d128", "max_num_seqs": 4, "max_model_len": 512, "num_blocks": 128, **kw}
    kw.setdefault("dtype", "bfloat16" if dev == "cuda" else "float32")
    e = LLMEngine(EngineConfig(**kw), device="cuda:0" if dev == "cuda" else "cpu")
    if dev == "cuda":
        e.warmup()
    return e


def prompt(n, seed):
    return torch.randint(3, 250, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def drain(e, seqs):
    while any(not s.finish_reason for s in seqs):
        e.step()
    return [s.output_ids for s in seqs]


# ---------------------------------------------------------------- the 8-bit cache

@pytest.mark.parametrize("dev", DEVICES)
def test_chunks_steps_and_mixed_steps(dev):
    """Prompts longer than a step's budget, arrivals while others decode, a shared prefix: the same sequences come out whether they run
    alone or together, and logits stay near those of the unrounded cache."""
    kw = dict(max_prefill_tokens=48, mixed_prefill_tokens=32)
    prompts = [prompt(100, 1), prompt(17, 2), prompt(100, 1)[:64] + prompt(30, 3), prompt(5, 4)]
    par = SamplingParams(max_tokens=12, **GREEDY)
    e = engine(dev, kv_cache_dtype="fp8", **kw)
    seqs = []
    for p in prompts:
        seqs.append(e.add_request(p, par))
        e.step()
        e.step()
    together = drain(e, seqs)
    assert all(len(o) == 12 for o in together)
    assert e.runner.n_steps.get("mixed", 0) > 0 and e.runner.n_steps["prefill_context_tokens"] > 0
    if dev == "cpu":  # fp32 rows: a sequence's pages do not depend on what runs beside it, only on where its prompt was cut
        alone = engine(dev, kv_cache_dtype="fp8", prefix_caching=False, **kw)
        for p, o in zip(prompts[1::2], together[1::2]):
            assert drain(alone, [alone.add_request(p, par)])[0] == o


@pytest.mark.parametrize("dev", DEVICES)
def test_logits_are_near_those_of_the_unrounded_cache(dev):
    """Step after step on the same tokens: an e4m3 number is off by at most half a step, 2^-4 relative - values by that, probabilities by no more
    where scores are of size 1 -, in each of two layers, whose sum with the residual stream the norms do not amplify: 2 * 2 * 2^-4 of the
    logits' norm."""
    p = prompt(60, 7)
    got = []
    for kind in ("auto", "fp8"):
        e = engine(dev, kv_cache_dtype=kind, keep_logits=True, pipeline=False)
        s = e.add_request(p, SamplingParams(max_tokens=20, **GREEDY))
        rows = []
        while not s.finish_reason:
            e.step()
            # (a replayed step's logits lie in its own buffer)
            rows.append((e.runner.last_logits[-1] if len(s.output_ids) == 1 else e.runner.d_logits[0]).float().cpu().clone())
            if got:
                s.output_ids[-1] = got[0][1][len(s.output_ids) - 1]  # the same tokens on both sides
        got.append((torch.stack(rows), list(s.output_ids)))
    a, b = got[0][0], got[1][0]
    assert a.shape == b.shape and float((a - b).norm() / a.norm()) <= 0.25
    assert not torch.equal(a[5:], b[5:])


def test_the_cache_takes_half_the_memory():
    a, b = engine("cpu", num_blocks=None, kv_cache_gb=0.01, dtype="bfloat16"), engine("cpu", num_blocks=None, kv_cache_gb=0.01, dtype="bfloat16", kv_cache_dtype="fp8")
    assert b.runner.num_blocks > 1.95 * a.runner.num_blocks
    assert b.runner.memory_report()["kv_cache_bytes"] <= 0.01 * (1 << 30)


def test_gpt2_heads_run_over_the_8_bit_cache():
    e = engine("cpu", model="gpt2-tiny", max_model_len=128, num_blocks=32, kv_cache_dtype="fp8", max_prefill_tokens=16)
    assert len(drain(e, [e.add_request(prompt(40, 3), SamplingParams(max_tokens=3, **GREEDY))])[0]) == 3


def test_refused_configurations():
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        engine("cpu", kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="head size"):
        engine("cpu", model="llama-tiny", kv_cache_dtype="fp8", model_overrides=dict(head_dim=32, n_heads=4, n_kv_heads=2))


# ---------------------------------------------------------------- controls

def oracle(e, ids, n, p):
    """Greedy under the controls, from whole forwards."""
    out = []
    for _ in range(n):
        x = _logits(e, ids + out).double()
        seen = sorted(set(ids + out))
        t = x[seen]
        x[seen] = torch.where(t > 0, t / p.repetition_penalty, t * p.repetition_penalty)
        for v in set(out):
            x[v] -= p.frequency_penalty * out.count(v) + p.presence_penalty
        for v, a in (p.logit_bias or {}).items():
            x[v] += a
        if p.allowed_token_ids is not None:
            keep = torch.full_like(x, float("-inf"))
            keep[list(p.allowed_token_ids)] = 0
            x = x + keep
        out.append(int(x.argmax()))
    return out


PARAMS = [dict(repetition_penalty=1.7), dict(presence_penalty=1.5, frequency_penalty=0.8), dict(logit_bias={11: 4.0, 12: -100.0, 13: 3.5}),
          dict(allowed_token_ids=(5, 9, 77, 200), repetition_penalty=1.3), dict(frequency_penalty=-0.5), {}]


@pytest.mark.parametrize("pipeline", [True, False])
def test_controlled_answers_are_the_definitions(pipeline):
    """Together, on four sequence slots, with chunks, mixed and pipelined steps: each answer is what whole forwards and the definition give."""
    e = engine("cpu", logit_controls=True, pipeline=pipeline, max_prefill_tokens=24, mixed_prefill_tokens=16)
    prompts = [prompt(30 + 7 * i, 20 + i) for i in range(len(PARAMS))]
    pars = [SamplingParams(max_tokens=8, **GREEDY, **k) for k in PARAMS]
    seqs = [e.add_request(p, q) for p, q in zip(prompts, pars)]
    got = drain(e, seqs)
    for ids, p, o in zip(prompts, pars, got):
        assert o == oracle(e, ids, 8, p)


def _logits(e, ids):
    """The last row's logits of a whole forward without a cache."""
    from k8s_llm_monitor_amd.models.llama import AttnMeta
    t = torch.tensor(ids, dtype=torch.int32)
    meta = AttnMeta(is_prefill=True, positions=torch.arange(len(ids), dtype=torch.int32), slot_mapping=torch.full((len(ids),), -1, dtype=torch.int32),
                    cu_seqlens=torch.tensor([0, len(ids)], dtype=torch.int32), logits_idx=torch.tensor([len(ids) - 1]))
    return e.model.forward(t, meta, None)[0].float()


def test_more_requests_than_slots_and_preemption():
    """Twelve controlled requests on three sequence slots and few pages: control slots come back, preempted sequences get new ones."""
    e = engine("cpu", logit_controls=True, max_num_seqs=3, num_blocks=14, max_model_len=96, prefix_caching=False)
    pars = [SamplingParams(max_tokens=30, **GREEDY, **PARAMS[i % len(PARAMS)]) for i in range(12)]
    prompts = [prompt(40 + i, 50 + i) for i in range(12)]
    got = drain(e, [e.add_request(p, q) for p, q in zip(prompts, pars)])
    assert e.counters["preemptions"] > 0
    for i in (0, 3, 4, 9):
        assert got[i] == oracle(e, prompts[i], 30, pars[i])


@pytest.mark.gpu
def test_controlled_answers_on_the_gpu():
    """Captured, pipelined steps: allowed tokens only, no token twice under a presence penalty that outweighs every logit, a bias that
    decides, beside a row without controls that answers as in an engine without them."""
    plain = engine("cuda")
    e = engine("cuda", logit_controls=True)
    allowed = tuple(range(40, 60))
    ks = [dict(allowed_token_ids=allowed, presence_penalty=1e4), {}, dict(logit_bias={123: 1e4}), dict(presence_penalty=1e4)]
    prompts = [prompt(50, 80 + i) for i in range(4)]
    got = drain(e, [e.add_request(p, SamplingParams(max_tokens=16, **GREEDY, **k)) for p, k in zip(prompts, ks)])
    assert set(got[0]) <= set(allowed) and len(set(got[0])) == 16
    assert got[1] == drain(plain, [plain.add_request(prompts[1], SamplingParams(max_tokens=16, **GREEDY))])[0]
    assert got[2] == [123] * 16 and len(set(got[3])) == 16


@pytest.mark.gpu
def test_both_together_on_the_gpu():
    e = engine("cuda", logit_controls=True, kv_cache_dtype="fp8", max_prefill_tokens=64)
    seqs = [e.add_request(prompt(90, 90 + i), SamplingParams(max_tokens=24, temperature=0.8, top_k=20, ignore_eos=True, allowed_token_ids=tuple(range(i, 250, 3)),
                                                             repetition_penalty=1.1)) for i in range(3)]
    for i, o in enumerate(drain(e, seqs)):
        assert len(o) == 24 and all(t % 3 == i for t in o)


def test_refused_requests():
    e = engine("cpu")
    with pytest.raises(ValueError, match="logit_controls"):
        e.add_request([5, 6], SamplingParams(presence_penalty=1.0))
    e = engine("cpu", logit_controls=True, max_logit_bias=2)
    V = e.model_cfg.vocab_size
    for bad in (dict(repetition_penalty=0.0), dict(logit_bias={V: 1.0}), dict(logit_bias={1: 1.0, 2: 1.0, 3: 1.0}), dict(allowed_token_ids=()),
                dict(allowed_token_ids=(-1,)), dict(frequency_penalty=float("nan"))):
        with pytest.raises(ValueError):
            e.add_request([5, 6], SamplingParams(**bad))
    assert not e.has_work()
    svc = EngineService(e)
    try:
        with pytest.raises(ValueError):
            svc.submit([5, 6], SamplingParams(logit_bias={V: 1.0})).result(timeout=30)
        assert svc.submit([5, 6], SamplingParams(max_tokens=2, **GREEDY, logit_bias={7: 1e4})).result(timeout=60)[1].output_ids == [7, 7]
    finally:
        svc.close()


def test_chat_requests_have_them():
    """POST /v1/chat/completions: presence_penalty, frequency_penalty, logit_bias reach a backend that takes them; 400 for what it refuses."""
    from k8s_llm_monitor_amd.monitor.server import MonitorApp, _chat_controls
    assert _chat_controls({"presence_penalty": 1, "logit_bias": {"7": -2}}) == {"presence_penalty": 1.0, "logit_bias": {7: -2.0}}
    for bad in ({"presence_penalty": "x"}, {"logit_bias": {"a": 1}}, {"logit_bias": [1]}, {"frequency_penalty": True}):
        with pytest.raises(Exception) as err:
            _chat_controls(bad)
        assert err.value.code == 400

    class Backend:
        takes_controls = True

        def generate(self, prompt, max_tokens=None, temperature=None, top_p=None, controls=None):
            if controls and 9 in controls.get("logit_bias", {}):
                raise ValueError("token 9")
            return {"text": json.dumps(controls), "model": "m"}

    class Analysis:
        backend = Backend()

        def fit_chat(self, parts, mt):
            return "\n".join(parts)

    app = MonitorApp.__new__(MonitorApp)
    app.analysis = Analysis()
    app._bounded = lambda fn: fn()
    ask = lambda **k: app.chat_completions("POST", json.dumps({"messages": [{"role": "user", "content": "hi"}], **k}).encode(), {})  # noqa: E731
    text = lambda r: json.loads(r.body)["choices"][0]["message"]["content"]  # noqa: E731
    assert json.loads(text(ask(frequency_penalty=0.5))) == {"frequency_penalty": 0.5}
    assert text(ask()) == "null"
    with pytest.raises(Exception) as err:
        ask(logit_bias={"9": 1})
    assert err.value.code == 400
    Backend.takes_controls = False
    assert text(ask(frequency_penalty=0.5)) == "null"


@pytest.mark.parametrize("field", [{"presence_penalty": 10 ** 400}, {"logit_bias": {"1": -10 ** 400}}])
def test_chat_numbers_of_hundreds_of_digits_are_bad_requests(field):
    from k8s_llm_monitor_amd.monitor.server import _chat_controls
    with pytest.raises(Exception) as err:
        _chat_controls(json.loads(json.dumps(field)))
    assert err.value.code == 400


# ---------------------------------------------------------------- one rule for every prompt

def first_logits(e, s, steps=40):
    """The logits that a prompt's first token is taken from."""
    for _ in range(steps):
        e.step()
        if s.output_ids:
            return e.runner.last_logits[-1].float().cpu().clone()
    raise AssertionError("no token")


def held_codes(e, s, n):
    """The key codes of a sequence's first n tokens, every layer."""
    pages = torch.tensor(s.block_table[: n // 16])
    return e.runner.k_cache.view(torch.uint8)[:, pages.to(e.runner.k_cache.device)].cpu()


def test_a_prompt_answers_alike_alone_beside_others_and_in_chunks():
    """fp32 rows: beside a prompt whose prefix is cached, and cut into chunks (at a page's border and inside one), a prompt's logits and pages are
    what they are alone.  The matrix products' row counts differ, so rows do by a few steps of 2^-24, and now and then a code whose value lies that near
    to the middle of two (of a thousand codes fewer than one); 2^-10 of the norm is far above both, and thirty times below what attending unrounded rows makes."""
    kw = dict(kv_cache_dtype="fp8", keep_logits=True, pipeline=False)
    p, shared = prompt(60, 7), prompt(64, 8)
    par = SamplingParams(max_tokens=4, **GREEDY)
    got = []
    for how in ("alone", "beside", "chunks of 48", "chunks of 40"):
        e = engine("cpu", **kw, **({"max_prefill_tokens": int(how[-2:])} if how[:6] == "chunks" else {}))
        if how == "beside":
            drain(e, [e.add_request(shared + prompt(3, 9), par)])
            e.add_request(shared + prompt(30, 10), par)
        s = e.add_request(p, par)
        got.append((first_logits(e, s), held_codes(e, s, len(p))))
        if how == "beside":
            assert e.runner.n_steps["prefill_context_tokens"] >= 64
    for logits, codes in got[1:]:
        assert float((logits - got[0][0]).norm() / got[0][0].norm()) <= 2.0 ** -10
        assert float((codes != got[0][1]).float().mean()) <= 1e-3


@pytest.mark.parametrize("dev", DEVICES)
def test_whole_prompts_attend_the_pages(dev, monkeypatch):
    """No step over the 8-bit cache attends unrounded rows; a step without block tables is refused."""
    from k8s_llm_monitor_amd import ops
    from k8s_llm_monitor_amd.models.llama import AttnMeta
    e = engine(dev, kv_cache_dtype="fp8")
    calls = []
    whole, pages = ops.flash_prefill, ops.flash_prefill_kv8
    monkeypatch.setattr(ops, "flash_prefill", lambda *a, **k: calls.append("rows") or whole(*a, **k))
    monkeypatch.setattr(ops, "flash_prefill_kv8", lambda *a, **k: calls.append("pages") or pages(*a, **k))
    drain(e, [e.add_request(prompt(n, n), SamplingParams(max_tokens=3, **GREEDY)) for n in (1, 20, 70)])
    assert calls and set(calls) == {"pages"}
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=e.runner.device)  # noqa: E731
    meta = AttnMeta(is_prefill=True, positions=i32(0, 1), slot_mapping=i32(-1, -1), cu_seqlens=i32(0, 2), logits_idx=i32(1).long())
    with pytest.raises(ValueError, match="block_tables"):
        e.model.forward(i32(5, 6), meta, e.runner.kv)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("top_p", [1.0, 0.9])
def test_an_infinite_bias_beside_an_ordinary_request(dev, top_p):
    """Sampled at a temperature: the biased row takes its token at every step, the other request finishes."""
    e = engine(dev, logit_controls=True)
    par = dict(max_tokens=6, temperature=0.7, top_p=top_p, ignore_eos=True)
    got = drain(e, [e.add_request(prompt(20, 1), SamplingParams(logit_bias={7: float("inf")}, **par)), e.add_request(prompt(30, 2), SamplingParams(**par))])
    assert got[0] == [7] * 6 and len(got[1]) == 6


def test_requests_that_allow_no_token_are_refused():
    e = engine("cpu", logit_controls=True)
    out = float("-inf")
    for bad in (dict(allowed_token_ids=(5,), logit_bias={5: out}), dict(allowed_token_ids=(5, 6, 5), logit_bias={5: out, 6: out, 9: 1.0})):
        with pytest.raises(ValueError, match="allowed"):
            e.add_request([5, 6], SamplingParams(**bad))
    few = engine("cpu", logit_controls=True, max_logit_bias=2000)  # (the vocabulary has 1024)
    with pytest.raises(ValueError, match="allowed"):
        few.add_request([5, 6], SamplingParams(logit_bias=dict.fromkeys(range(few.model_cfg.vocab_size), out)))
    s = e.add_request([5, 6], SamplingParams(max_tokens=3, temperature=0.9, ignore_eos=True, allowed_token_ids=(5, 6), logit_bias={5: out}))
    assert drain(e, [s])[0] == [6] * 3


@pytest.mark.parametrize("bias", [[], 0, False, "", "7", {"7": "5"}, {"7": "inf"}, {"7": True}, {"7": None}, {"07": 1}, {" 7": 1}, {"1_0": 1}, {"-1": 1}, {"7.0": 1}])
def test_chat_biases_of_another_type_are_bad_requests(bias):
    from k8s_llm_monitor_amd.monitor.server import _chat_controls
    with pytest.raises(Exception) as err:
        _chat_controls({"logit_bias": bias})
    assert err.value.code == 400
    assert _chat_controls({"logit_bias": {}}) == _chat_controls({"logit_bias": None}) == {}


# ---------------------------------------------------------------- whole engines, by what they leave in their pages

def held(e, s):
    """What a sequence's pages stand for: [layers, 2, tokens, Hkv, D] of the tokens whose rows have run."""
    from k8s_llm_monitor_amd.ops import KV8
    from k8s_llm_monitor_amd.ops.kv8 import gather_kv8
    table, n = torch.tensor(s.block_table), s.num_tokens - 1
    rows = [gather_kv8(KV8(*(t.cpu() for t in e.runner.kv[i])), table, n) for i in range(len(e.runner.kv))]
    return torch.stack([torch.stack(r) for r in rows])


def run_forced(e, arrivals, steps=12):
    """Requests that arrive every other step, each fed tokens of its own at every step: what their pages hold one token before the end."""
    par = SamplingParams(max_tokens=steps, **GREEDY)
    seqs, out = [], {}
    while len(out) < len(arrivals):
        if len(seqs) < len(arrivals):
            seqs.append(e.add_request(arrivals[len(seqs)], par))
        for _ in range(2):
            e.step()
            for i, s in enumerate(seqs):
                if s.output_ids and not s.finish_reason:
                    s.output_ids[-1] = 3 + (31 * i + 7 * len(s.output_ids)) % 240
                    if len(s.output_ids) == steps - 1:
                        out[i] = held(e, s)
    return [out[i] for i in range(len(arrivals))]


@pytest.mark.parametrize("dev", DEVICES)
def test_pages_of_chunks_mixed_steps_and_prefix_hits(dev):
    """Together, with chunks, mixed steps and a cached prefix, sequences leave in their pages what each leaves alone, whole.  Rows of other steps go through
    other matrix kernels: at most 12 roundings a layer of half a bf16 step (2^-9) in two layers, 0.047 of the norm, and where rows differ by that a code in
    32 is the neighbouring one, 2^-3 off, 0.022 of the norm.  (fp32 rows: 2^-10 as above.)  A wrong page or position is off by the norm itself."""
    kw = dict(kv_cache_dtype="fp8", pipeline=False)
    arrivals = [prompt(100, 1), prompt(17, 2), prompt(100, 1)[:64] + prompt(30, 3), prompt(5, 4)]
    e = engine(dev, max_prefill_tokens=48, mixed_prefill_tokens=32, **kw)
    together = run_forced(e, arrivals)
    assert e.runner.n_steps.get("mixed", 0) > 0 and e.runner.n_steps["prefill_context_tokens"] >= 64
    for i, p in enumerate(arrivals):
        alone = run_forced(engine(dev, prefix_caching=False, **kw), [arrivals[j] if j == i else [3] for j in range(len(arrivals))])[i]
        assert alone.shape == together[i].shape
        for a, b in zip(alone.flatten(0, 1), together[i].flatten(0, 1)):
            assert float((a - b).norm() / a.norm()) <= (0.07 if dev == "cuda" else 2.0 ** -10)


def _tp_worker(rank, world, port, q):
    import os
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
    torch.set_num_threads(2)
    from k8s_llm_monitor_amd.engine.runner import ModelRunner
    from k8s_llm_monitor_amd.parallel.state import ParallelState, destroy, init_parallel
    try:
        ps = init_parallel(tp_size=world, device="cpu")
        micro = []
        # steps of several prompts in two micro-batches, however few their rows
        ModelRunner._micro_split = staticmethod(lambda cu, nd, min_rows=0: micro.append(1) or 1 if len(cu) > 2 and not nd else 0)
        cfg = EngineConfig(model="llama-tiny-d128", max_num_seqs=4, max_model_len=512, num_blocks=128, use_graphs=False, dtype="float32",
                           kv_cache_dtype="fp8", keep_logits=True, max_prefill_tokens=200)
        shared = prompt(64, 1)
        asks = [[prompt(100, 5), prompt(17, 2), shared], [shared + prompt(30, 3), prompt(5, 4)], [prompt(300, 6)]]

        def drive(e):
            par, got = SamplingParams(max_tokens=3, **GREEDY), []
            for ask in asks:
                seqs = [e.add_request(p, par) for p in ask]
                while not all(s.output_ids for s in seqs):
                    e.step()
                got.append(e.runner.last_logits.float().clone())
                drain(e, seqs)
            return got
        e = LLMEngine(cfg, device="cpu", pstate=ps)
        got = None
        if ps.tp_rank == 0:
            got = drive(e)
            e.stop_workers()
        else:
            e.worker_loop()
        e.bus.close()
        n = len(micro)
        if got is not None:
            want = drive(LLMEngine(cfg, device="cpu", pstate=ParallelState()))
            q.put((rank, [float((a - b).norm() / b.norm()) for a, b in zip(got, want)], n))
        else:
            q.put((rank, [0.0], n))
        destroy()
    except Exception as err:  # noqa: BLE001
        import traceback
        q.put((rank, repr(err) + traceback.format_exc(), 0))


@pytest.mark.parametrize("world", [2, 4])
def test_tensor_parallel_engines(world):
    """Heads split over ranks (4 ranks: kv heads on two each), micro-batches, chunks, a prefix hit: the prompts' logits are those of one rank (the bound: as
    above, the sums over ranks are rounded in another order)."""
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_tp_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = [q.get(timeout=300) for _ in procs]
    for p in procs:
        p.join(60)
    for rank, errs, micro in res:
        assert not isinstance(errs, str), errs
        assert max(errs) <= 2.0 ** -10 and micro > 0


def _on_cpu(x):
    if isinstance(x, torch.Tensor):
        return x.cpu()
    if isinstance(x, dict):
        return {k: _on_cpu(v) for k, v in x.items()}
    return type(x)(map(_on_cpu, x)) if isinstance(x, (list, tuple)) and type(x) in (list, tuple) else x


@pytest.mark.gpu
def test_gpt2_pages_on_the_gpu():
    """GPT-2's heads (64 dims, no rotation, biases): with the same weights, the GPU's pages are the CPU's.  The bound: as above."""
    kw = dict(model="gpt2-tiny", max_model_len=128, num_blocks=64, kv_cache_dtype="fp8", max_prefill_tokens=16, pipeline=False)
    arrivals = [prompt(40, 3), prompt(7, 4), prompt(20, 5)]
    e, c = engine("cuda", **kw), engine("cpu", dtype="bfloat16", **kw)
    for name in ("embed", "pos_embed", "final_norm", "layers", "lm_head"):
        if hasattr(e.model, name):
            setattr(c.model, name, _on_cpu(getattr(e.model, name)))
    for a, b in zip(run_forced(e, arrivals), run_forced(c, arrivals)):
        for x, y in zip(a.flatten(0, 1), b.flatten(0, 1)):
            assert float((x - y).norm() / y.norm()) <= 0.07
