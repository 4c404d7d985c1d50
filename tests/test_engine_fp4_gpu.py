"""The engine with MXFP4 projections: the model's step against the same step on the ops' fp64 statements, graph
replay against eager steps, and the checkpoint families it serves (dense, Shadow Residual, experts)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ALL = ("q", "k", "v", "o", "gate", "up", "down")
# family: (LoRA targets, extra composition arguments)
FAMILIES = {
    "dense": (ALL, {}),
    "attention_lora": (("q", "k", "v"), {}),
    "shadow": (("q", "o", "gate", "up", "down"), dict(cross_rank=16, std_b=0.03)),
    "experts": (ALL, dict(num_local_experts=8, num_experts_per_tok=2, intermediate_size=256,
                          shared_intermediate_size=512)),
}


@pytest.fixture(scope="module", params=list(FAMILIES))
def family_dir(request, tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA")
    from granite_switch_b200.composer.synthetic import compose_synthetic

    d = str(tmp_path_factory.mktemp("fp4_" + request.param))
    targets, extra = FAMILIES[request.param]
    compose_synthetic(d, "tiny", num_adapters=3, rank=8, targets=targets, seed=4, dtype=torch.float32,
                      invocation_len=4, alpha=16.0, num_hidden_layers=2, **extra)
    return d


def _model(d, weight_dtype):
    from granite_switch_b200.checkpoint import load_state_dict
    from granite_switch_b200.config import GraniteSwitchConfig
    from granite_switch_b200.models.native import NativeGraniteSwitch

    cfg = GraniteSwitchConfig.from_pretrained(d)
    return cfg, NativeGraniteSwitch.from_state_dict(cfg, load_state_dict(d), torch.device("cuda", 0), max_tokens=1024,
                                                    num_kv_blocks=128, max_seqs=8, weight_dtype=weight_dtype)


def _prompts(cfg):
    g = torch.Generator().manual_seed(3)
    ids = lambda n: torch.randint(5, 900, (n,), generator=g).tolist()  # noqa: E731
    c = list(cfg.adapter_token_ids)
    return [ids(150) + [c[0]] + ids(3), ids(40), ids(9) + [c[2]] + ids(130), [c[1]] + ids(2)]


def _logits(cfg, model, forced, steps=3):
    """Logits of a prefill step and decode steps fed with ``forced`` tokens (filled with greedy ones when empty)."""
    from granite_switch_b200.engine.executor import NativeExecutor
    from granite_switch_b200.engine.kv_cache import BlockManager
    from granite_switch_b200.engine.llm_engine import HostRouter
    from granite_switch_b200.engine.request import Request, SamplingParams
    from granite_switch_b200.engine.scheduler import Scheduler

    ex, bm, router = NativeExecutor(model, 1024), BlockManager(128), HostRouter(cfg)
    sch = Scheduler(bm, 8, 1024, True, route_fn=router)
    for p in _prompts(cfg):
        sch.add(Request(p, SamplingParams(max_tokens=steps)))
    outs = []
    for step in range(steps):
        out = sch.schedule()
        _, logits = ex.compute_logits(out)
        outs.append(logits[:, : cfg.vocab_size].float().cpu())
        if len(forced) <= step:
            forced.append(outs[-1].argmax(-1).tolist())
        j = 0
        for c in out.chunks:
            r = c.req
            r.carry = router(r.all_ids[c.start:c.start + c.num_tokens], r.carry)
            r.num_computed = c.start + c.num_tokens
            bm.register_full_blocks(r)
            if c.needs_sample:
                r.output_ids.append(forced[step][j])
                j += 1
    return outs


class _Statements:
    """ops.gemm_fp4 with every kernel replaced by its fp64 statement (the outputs' types and buffers as the kernels')."""

    def __getattr__(self, name):
        from granite_switch_b200.ops import gemm_fp4 as F

        return getattr(F, name)

    @staticmethod
    def _masked(kw, m, cols):
        """The shrink output with the columns of adapters absent from a tile (never written) as zeros."""
        s, mask, na, rank = kw["s"].double(), kw["tile_mask"], kw["num_adapters"], kw["rank"]
        a = (torch.arange(s.shape[1], device=s.device) // rank) % na
        here = (mask[torch.arange(m, device=s.device) // 128][:, None] >> a) & 1
        return torch.where(here.bool(), s, 0.0)[:, :cols]

    def quantize_rows_mxfp4(self, x, *codes):
        from granite_switch_b200.ops import gemm_fp4 as F

        return F.quantize_rows_reference(x)

    def rmsnorm_mxfp4(self, x, w, eps, x4=None, sf=None, out=None):
        from granite_switch_b200.ops import elementwise as E
        from granite_switch_b200.ops import gemm_fp4 as F

        if out is not None:
            out.copy_(E.rmsnorm_reference(x, w, eps))
        v = x.double()
        return F.quantize_rows_reference(v * torch.rsqrt(v.square().mean(1, keepdim=True) + eps) * w.double())

    def _acc(self, x4, sfx, w4, sfw, kw):
        from granite_switch_b200.ops import gemm_fp4 as F

        if not kw:
            return F.mxfp4_product_reference(x4, sfx, w4, sfw)
        bounds = kw.get("slice_bounds")
        cols = kw["lb"].shape[1] * (len(bounds) - 1 if bounds else 1)
        return F.mxfp4_product_reference(x4, sfx, w4, sfw, s=self._masked(kw, x4.shape[0], cols), lb=kw["lb"],
                                         rank=kw["rank"], num_adapters=kw["num_adapters"], slice_bounds=bounds)

    def mxfp4_gemm(self, x4, sfx, w4, sfw, out, *, epi, scale, residual, **kw):
        v = self._acc(x4, sfx, w4, sfw, kw) * scale
        out.copy_((v + residual.double() if epi else v).to(out.dtype))
        return out

    def mxfp4_gemm_swiglu(self, x4, sfx, w4, sfw, a4=None, sf=None, act=None, **kw):
        from granite_switch_b200.ops import gemm_fp4 as F

        v = F.swiglu_reference(self._acc(x4, sfx, w4, sfw, kw))
        if act is not None:
            act.copy_(v.to(act.dtype))
        return F.quantize_rows_reference(v)


def test_step_matches_the_statements(family_dir, monkeypatch):
    """Kernels and fp64 statements differ by fp32 sums: a bf16 output now and then rounds to its neighbour (2^-8 of
    the value, one element in some thousands), and fewer still of those move a 4-bit code. Logits, sums over 256 such
    values, stay within 2% of their largest. Against the bf16 model the logits must be recognisably the same."""
    from granite_switch_b200._native import check_errors
    from granite_switch_b200.models import native

    cfg, model = _model(family_dir, "mxfp4")
    assert all(pl.w is None and pl.w4 is not None for lw in model.layers for pl in (lw.qkv, lw.o, lw.gu, lw.down))
    forced = []
    got = _logits(cfg, model, forced)
    check_errors(torch.device("cuda", 0))
    plain = _logits(cfg, _model(family_dir, "bfloat16")[1], forced)
    monkeypatch.setattr(native, "F4", _Statements())
    want = _logits(cfg, model, forced)
    for a, b, c in zip(got, want, plain):
        assert a.shape == b.shape and a.isfinite().all()
        assert (a - b).abs().max() <= 0.02 * b.abs().max(), float((a - b).abs().max() / b.abs().max())
        # 4-bit rounding moves a product by about 16% of its norm (two operands of 11%); random weights of
        # two layers leave the logits with a cosine above 0.9
        cos = torch.nn.functional.cosine_similarity(a.flatten(), c.flatten(), dim=0)
        assert cos > 0.9, float(cos)


def test_graph_replay_and_async_steps(family_dir):
    """Greedy tokens are the same from eager, graph-replayed and pipelined steps."""
    from granite_switch_b200.engine import LLM, EngineConfig, SamplingParams

    toks = []
    for graphs, asynch in ((False, False), (True, False), (True, True)):
        llm = LLM(family_dir, device="cuda:0",
                  engine_config=EngineConfig(max_num_seqs=8, max_num_batched_tokens=128, num_kv_blocks=128,
                                             max_model_len=512, use_cuda_graphs=graphs, async_scheduling=asynch,
                                             weight_dtype="mxfp4"))
        outs = llm.generate(_prompts(llm.config), SamplingParams(max_tokens=8))
        assert llm.engine.stats.device_errors == 0
        if graphs:
            assert llm.engine.executor.graph_replays > 0
        toks.append([o.output_ids for o in outs])
    assert toks[0] == toks[1] == toks[2]


def test_fp8_cache_and_random_weights():
    """4-bit weights beside an fp8 KV cache, weights drawn on the GPU."""
    from granite_switch_b200.composer.synthetic import base_config
    from granite_switch_b200.config import GraniteSwitchConfig
    from granite_switch_b200.engine import LLM, EngineConfig, SamplingParams

    base = base_config("tiny")
    na, v = 3, base["vocab_size"]
    cfg = dict(base, num_adapters=na, adapter_token_ids=list(range(v, v + na)), adapter_substitute_token_ids=[1] * na,
               adapter_ranks=[8] * na, max_lora_rank=8, lora_target_modules=["qkv_proj", "o_proj"],
               num_hidden_layers=base["num_hidden_layers"] + 2, vocab_size=v + na)
    llm = LLM(GraniteSwitchConfig(**cfg), device="cuda:0",
              engine_config=EngineConfig(max_num_seqs=4, max_num_batched_tokens=256, num_kv_blocks=64, max_model_len=512,
                                         kv_cache_dtype="fp8_e4m3", weight_dtype="mxfp4"),
              random_init=dict(lora_modules=("qkv", "o"), rank=8))
    outs = llm.generate([[5, 6, 7, v, 9, 10] * 8, [11, 12, v + 1, 13] * 5], SamplingParams(max_tokens=4))
    assert [len(o.output_ids) for o in outs] == [4, 4] and llm.engine.stats.device_errors == 0


def test_parallel_models_are_refused():
    from granite_switch_b200.models.native import NativeGraniteSwitch

    with pytest.raises(ValueError, match="one GPU"):
        NativeGraniteSwitch(None, torch.device("cuda", 0), 64, 8, tp_size=2, weight_dtype="mxfp4")
    with pytest.raises(ValueError, match="weight_dtype"):
        NativeGraniteSwitch(None, torch.device("cuda", 0), 64, 8, weight_dtype="int4")


@pytest.mark.parametrize("on", [False, True])
def test_programmatic_launch_switch_reaches_the_kernels(on):
    """An engine with 4-bit projections sets the launch kind of every kernel, the MXFP4 ones included."""
    from granite_switch_b200._native import native
    from granite_switch_b200.composer.synthetic import base_config
    from granite_switch_b200.config import GraniteSwitchConfig
    from granite_switch_b200.engine import LLM, EngineConfig, SamplingParams

    old = native().set_pdl(-1)
    try:
        llm = LLM(GraniteSwitchConfig(**base_config("tiny")), device="cuda:0",
                  engine_config=EngineConfig(max_num_seqs=2, max_num_batched_tokens=64, num_kv_blocks=32,
                                             max_model_len=128, weight_dtype="mxfp4", programmatic_launch=on),
                  random_init={})
        assert len(llm.generate([[5, 6, 7]], SamplingParams(max_tokens=2))[0].output_ids) == 2
        assert native().set_pdl(1) == int(on)
    finally:
        native().set_pdl(old)


def test_norms_are_rounded_once(family_dir, monkeypatch):
    """Every layer norm goes from fp32 to 4 bits in one kernel, in both streams of Shadow Residual: the bf16 RMSNorm
    runs for the final norm alone, and only the inputs of the o projections meet a quantiser of their own."""
    from granite_switch_b200.models import native

    cfg, model = _model(family_dir, "mxfp4")
    calls = dict(rmsnorm=0, rmsnorm_mxfp4=0, quantize_rows_mxfp4=0)

    def counted(module, name):
        fn = getattr(module, name)

        def call(*a, **kw):
            calls[name] += 1
            return fn(*a, **kw)

        monkeypatch.setattr(module, name, call)

    counted(native.E, "rmsnorm")
    counted(native.F4, "rmsnorm_mxfp4")
    counted(native.F4, "quantize_rows_mxfp4")
    steps, streams = 2, 2 if model.layers[0].cross is not None else 1
    _logits(cfg, model, [], steps=steps)
    n = steps * len(model.layers) * streams
    assert calls == dict(rmsnorm=steps, rmsnorm_mxfp4=2 * n, quantize_rows_mxfp4=n)
