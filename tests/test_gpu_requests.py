"""Requests of one batch that differ, through the model, the generation loops, the
decode graph and the Scheduler: adapters, penalties, biases, grammars and parameters of
their own, against the same requests computed alone and in plain torch."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import requests_ref as ref
from serving.adapters import AdapterSet, step_adapters
from serving.allocator import BlockAllocator
from serving.batch import build_batch_step
from serving.controls import RequestParams, TokenHistory, pack_mask
from serving.generation import generate_batched
from serving.graph_step import DecodeStepGraph
from serving.kv_pool import KVPool
from serving.layers import ModelConfig, SchedulerConfig
from serving.paged_meta import pack_batch_meta
from serving.paged_model import PagedTransformer
from serving.scheduler import Scheduler
from serving.sequence import Sequence

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 997


def make_model(dtype=torch.float32, d_model=128, heads=4, seed=0):
    cfg = ModelConfig(vocab_size=VOCAB, d_model=d_model, num_layers=3, num_heads=heads,
                      num_kv_heads=1, max_seq_len=256, dtype=dtype)
    torch.manual_seed(seed)
    return PagedTransformer(cfg).to(DEV, dtype).eval(), cfg


def adapter_state(model, seed, rank, skip=()):
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, mod in model.named_modules():
        if isinstance(mod, torch.nn.Linear) and name != "lm_head" and not any(
                s in name for s in skip):
            out[name + ".lora_A.weight"] = torch.randn(rank, mod.in_features, generator=g) \
                * mod.in_features ** -0.5
            out[name + ".lora_B.weight"] = torch.randn(mod.out_features, rank, generator=g) * 0.3
    return out


def merged(model, cfg, state, scale):
    """The model with the adapter's products added to its weights."""
    other = PagedTransformer(cfg).to(DEV, cfg.dtype).eval()
    other.load_state_dict(model.state_dict())
    mods = dict(other.named_modules())
    with torch.no_grad():
        for key, a in state.items():
            if ".lora_A." in key:
                name = key.split(".lora_A.")[0]
                b = state[name + ".lora_B.weight"]
                mods[name].weight += (scale * b.double() @ a.double()).to(DEV, cfg.dtype)
    return other


def pool_of(cfg, blocks=64, dtype=None):
    return KVPool(cfg.num_layers, 16, blocks, 1, cfg.head_dim, dtype or cfg.dtype, DEV)


def prompts_of(lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in lens]


@pytest.fixture(scope="module")
def served():
    model, cfg = make_model()
    weights = AdapterSet(model, 3, 16)
    states = [adapter_state(model, 1, 16), adapter_state(model, 2, 5, skip=("k_proj", "up_proj"))]
    weights.load(0, states[0], 0.5)
    weights.load(2, states[1], 1.0)
    models = {-1: model, 0: merged(model, cfg, states[0], 0.5), 1: model,
              2: merged(model, cfg, states[1], 1.0)}
    return model, cfg, weights, models


def test_logits_of_each_request_are_its_merged_models(served):
    """A ragged prompt step, then a decode step. fp32: the sums of both sides differ by
    rounding alone, some 1e-6 a layer of logits of the order of one."""
    model, cfg, weights, models = served
    lens, ids = [7, 1, 33, 20, 64], [0, -1, 2, 1, 0]
    seqs, alloc, pool = [], BlockAllocator(64), pool_of(cfg)
    for n, p in enumerate(prompts_of(lens)):
        seqs.append(Sequence(n, p, 16))
        seqs[-1].ensure_blocks(alloc)
    batch = build_batch_step([(s, s.token_ids) for s in seqs], DEV)
    got = model.forward_batch(batch, pool, weights, ids)
    alone_pools = [pool_of(cfg) for _ in seqs]
    for n, s in enumerate(seqs):
        want = models[ids[n]].forward_batch(build_batch_step([(s, s.token_ids)], DEV),
                                            alone_pools[n])
        assert torch.allclose(got[n], want[0], rtol=1e-4, atol=1e-4), n
    for s in seqs:
        s.append_token(11)
        s.ensure_blocks(alloc)
    got = model.forward_batch(build_batch_step([(s, [11]) for s in seqs], DEV), pool, weights, ids)
    for n, s in enumerate(seqs):
        want = models[ids[n]].forward_batch(build_batch_step([(s, [11])], DEV), alone_pools[n])
        assert torch.allclose(got[n], want[0], rtol=1e-4, atol=1e-4), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_requests_without_an_adapter_keep_their_bits(dtype):
    model, cfg = make_model(dtype, 256, 4)
    weights = AdapterSet(model, 2, 8)
    weights.load(1, adapter_state(model, 3, 8), 1.0)
    prompts, alloc = prompts_of([5, 9, 30, 2]), BlockAllocator(64)
    seqs = [Sequence(n, p, 16) for n, p in enumerate(prompts)]
    for s in seqs:
        s.ensure_blocks(alloc)
    pools = pool_of(cfg), pool_of(cfg)
    ids = [-1, 1, -1, 1]
    for step in range(3):
        new = [s.token_ids if step == 0 else s.token_ids[-1:] for s in seqs]
        batch = build_batch_step(list(zip(seqs, new)), DEV)
        plain = model.forward_batch(batch, pools[0])
        mixed = model.forward_batch(batch, pools[1], weights, ids)
        assert torch.equal(plain[0], mixed[0]) and torch.equal(plain[2], mixed[2])
        assert not torch.equal(plain[1], mixed[1])
        assert torch.equal(model.forward_batch(batch, pools[0], weights, [-1] * 4), plain)
        for s in seqs:
            s.append_token(17 + step)
            s.ensure_blocks(alloc)


def test_generate_batched_with_adapters(served):
    model, cfg, weights, models = served
    prompts, ids = prompts_of([12, 3, 40, 8]), [2, 0, -1, 0]
    got = generate_batched(model, prompts, 16, pool_of(cfg), BlockAllocator(64),
                           adapters=weights, adapter_ids=ids)
    for p, i, toks in zip(prompts, ids, got):
        assert toks == generate_batched(models[i], [p], 16, pool_of(cfg), BlockAllocator(64))[0]


def test_decode_graph_with_adapters(served):
    model, cfg, weights, models = served
    prompts, ids = prompts_of([12, 3, 40, 8]), [2, 0, -1, 0]
    want = generate_batched(model, prompts, 9, pool_of(cfg), BlockAllocator(64),
                            adapters=weights, adapter_ids=ids)
    alloc, pool = BlockAllocator(64), pool_of(cfg)
    seqs = [Sequence(n, p, 16) for n, p in enumerate(prompts)]
    for s in seqs:
        s.ensure_blocks(alloc)
    first = model.forward_batch(build_batch_step([(s, s.token_ids) for s in seqs], DEV), pool,
                                weights, ids).argmax(1)
    for s, t in zip(seqs, first.tolist()):
        s.append_token(t)
        s.block_table.extend(alloc.allocate_n(1))  # room to grow
    batch = build_batch_step([(s, s.token_ids[-1:]) for s in seqs], DEV)
    meta = pack_batch_meta(batch.block_tables, batch.query_start_loc, batch.positions, 4, DEV, 16)
    step = step_adapters(weights, ids, [0, 1, 2, 3, 4], DEV)
    saved = [t.clone() for t in (meta.positions, meta.start_pos, meta.seq_lens)]
    graph = DecodeStepGraph(model, pool, meta, first, warmup=1, adapters=step)
    # the warm-up steps ran on this state: put it back
    for t, s in zip((meta.positions, meta.start_pos, meta.seq_lens), saved):
        t.copy_(s)
    graph.ids.copy_(first)
    got = [first.tolist()] + [graph.replay().tolist() for _ in range(8)]
    assert [list(r) for r in zip(*got)] == want


class Words:
    """A grammar for the tests: a cycle of states, each allowing its own tokens."""

    def __init__(self, allowed):
        self.allowed, self.state, self.took = allowed, 0, []

    def mask(self):
        a = torch.zeros(VOCAB, dtype=torch.bool)
        a[self.allowed[self.state]] = True
        return pack_mask(a)

    def advance(self, token):
        assert token in self.allowed[self.state]
        self.took.append(token)
        self.state = (self.state + 1) % len(self.allowed)


def alone(model, cfg, prompt, n, p, allowed=None):
    """Greedy tokens of one request by the restated controls on the model's logits."""
    seq, alloc, pool = Sequence(0, prompt, 16), BlockAllocator(64), pool_of(cfg)
    out, new, state = [], seq.token_ids, 0
    for _ in range(n):
        seq.ensure_blocks(alloc)
        row = model.forward_batch(build_batch_step([(seq, new)], DEV), pool)[0]
        ok = None
        if allowed is not None:
            ok = np.zeros(VOCAB, dtype=bool)
            ok[allowed[state]] = True
            state = (state + 1) % len(allowed)
        row = ref.control(row.double().cpu().numpy(), seq.token_ids, len(prompt),
                          p.repetition_penalty, p.presence_penalty, p.frequency_penalty,
                          list(p.logit_bias.items()), ok)
        top = np.sort(row)[-2:]
        assert top[1] - top[0] > 1e-4  # a choice that rounding does not turn
        out.append(int(row.argmax()))
        seq.append_token(out[-1])
        new = out[-1:]
    return out


@pytest.mark.parametrize("budget", [None, 24])
def test_scheduler_serves_requests_that_differ(served, budget):
    """Chunked prompts and preemption (budget) among them."""
    model, cfg, weights, models = served
    prompts = prompts_of([20, 24, 18, 30, 5])
    cycles = [[3, 5, 7, 900], [10, 11, 996]]
    params = [
        RequestParams(temperature=0, repetition_penalty=1.3, adapter=0),
        RequestParams(temperature=0, presence_penalty=0.4, frequency_penalty=0.2,
                      logit_bias={5: 1.5, 17: -100.0}),
        None,
        RequestParams(temperature=0, adapter=2, grammar=Words(cycles), frequency_penalty=0.3),
        RequestParams(temperature=1.0, top_k=1, min_p=0.5, adapter=0),
    ]
    n = 40 if budget else 14
    want = []
    for p, r in zip(prompts, params):
        q = r or RequestParams()
        want.append(alone(models[q.adapter], cfg, p, n, q, cycles if q.grammar else None))
    nb = 10 if budget else 64
    sc = SchedulerConfig(max_num_seqs=5, max_num_batched_tokens=budget,
                         enable_chunked_prefill=True,
                         cudagraph_batch_sizes=[1, 2]) if budget else None
    alloc = BlockAllocator(nb)
    sched = Scheduler(model, pool_of(cfg, nb), alloc, SimpleNamespace(eos_token_id=-1),
                      block_size=16, temperature=1.0, top_k=1, top_p=1.0, sched_cfg=sc,
                      adapters=weights)
    for p, r in zip(prompts, params):
        sched.add_request(p, n, params=r)
    got, steps = {}, 0
    while sched.running or sched.waiting:
        for sid, tok, done in sched.step():
            got.setdefault(sid, []).append(tok)
        steps += 1
        assert steps < 2000
    assert (sched.num_preemptions > 0) == (budget is not None)
    assert [got[i] for i in range(5)] == want
    assert params[3].grammar.took == want[3][:-1]
    assert alloc.num_free == alloc.num_usable and not sched._history._row


def test_scheduler_refusals(served):
    model, cfg, weights, _ = served
    sched = Scheduler(model, pool_of(cfg), BlockAllocator(64), SimpleNamespace(eos_token_id=-1))
    with pytest.raises(ValueError, match="no adapter 0"):
        sched.add_request([1], 2, params=RequestParams(adapter=0))
    sched.adapters = weights
    with pytest.raises(ValueError, match="no adapter 3"):
        sched.add_request([1], 2, params=RequestParams(adapter=3))
    # a grammar that leaves nothing
    none = SimpleNamespace(mask=lambda: torch.zeros(-(-VOCAB // 32), dtype=torch.int32),
                           advance=lambda t: None)
    sched.add_request([1, 2], 2, params=RequestParams(grammar=none))
    with pytest.raises(ValueError, match="no token left"):
        sched.step()
    batch = SimpleNamespace(block_tables=[[1]], query_start_loc=[0, 1], positions=[0],
                            input_ids=torch.tensor([1], device=DEV))
    with pytest.raises(ValueError, match="needs an AdapterSet"):
        model.forward_batch(batch, pool_of(cfg), None, [0])
    with pytest.raises(ValueError, match="adapter 5 of 3"):
        model.forward_batch(batch, pool_of(cfg), weights, [5])
    with pytest.raises(ValueError, match="adapter ids"):
        model.forward_batch(batch, pool_of(cfg), weights, [0, 1])
    with pytest.raises(ValueError, match="adapter_ids"):
        generate_batched(model, [[1]], 2, pool_of(cfg), BlockAllocator(8), adapters=weights,
                         adapter_ids=[0, 0])


def test_a_request_that_no_step_could_serve_is_refused_when_it_is_added(served):
    model, cfg, _, _ = served
    sched = Scheduler(model, pool_of(cfg), BlockAllocator(64), SimpleNamespace(eos_token_id=-1))
    with pytest.raises(ValueError, match="outside the vocabulary"):
        sched.add_request([1], 2, params=RequestParams(logit_bias={VOCAB: 1.0}))
    with pytest.raises(ValueError, match="infinite logit"):
        sched.add_request([1], 2, params=RequestParams(logit_bias={1: 3e38}))
    sched.add_request([1], 3, params=RequestParams(logit_bias={VOCAB - 1: -float("inf")}))
    short = SimpleNamespace(mask=lambda: torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="words"):
        sched.add_request([1], 2, params=RequestParams(grammar=short))
    words = Words([[3, 5], [4]])
    sched.add_request([1, 2], 3, params=RequestParams(grammar=words))
    with pytest.raises(ValueError, match="another request"):  # waiting
        sched.add_request([3], 3, params=RequestParams(grammar=words))
    sched.step()
    with pytest.raises(ValueError, match="another request"):  # running
        sched.add_request([3], 3, params=RequestParams(grammar=words, temperature=0))
    while sched.running or sched.waiting:
        sched.step()
    sched.add_request([3], 3, params=RequestParams(grammar=words))  # that one is done


def test_a_set_loads_all_of_an_adapter_or_nothing(served):
    model, _, _, _ = served
    few = AdapterSet(model, 1, 4)
    state = adapter_state(model, 1, 4)
    state["layers.2.mlp.down_proj.lora_B.weight"] = torch.zeros(128, 3)
    with pytest.raises(ValueError, match="are not"):
        few.load(0, state)
    with pytest.raises(IndexError):
        few.load(1, adapter_state(model, 1, 4))
    assert not any(w.a.any() or w.b.any() or w.scales.any()
                   for ws in few.layers for w in ws.values())


def test_adapter_set_names(served):
    model, cfg, _, _ = served
    few = AdapterSet(model, 1, 4, projections=("qkv",))
    state = adapter_state(model, 1, 4)
    with pytest.raises(ValueError, match="no projection of this set"):
        few.load(0, state)
    few.load(0, {k: v for k, v in state.items() if "_proj" in k and "attn" in k})
    with pytest.raises(ValueError, match="without the other"):
        few.load(0, {"layers.0.attn.q_proj.lora_A.weight": torch.zeros(4, 128)})
    with pytest.raises(ValueError, match="no projection"):
        AdapterSet(model, 1, 4, projections=("lm_head",))
    few.clear(0)
    assert not few.layers[0]["qkv"].a.any()


@pytest.mark.parametrize("device", ["cpu", DEV])
def test_token_history(device):
    h = TokenHistory(device)
    tokens, lens, prompts = h.rows([4])
    assert lens.tolist() == [0] and prompts.tolist() == [0]
    for key in range(20):  # past the first rows
        h.put(key, list(range(key)), key // 2)
    h.append(3, 77)
    h.append(19, 5)
    h.append(3, 78)
    tokens, lens, prompts = h.rows([3, 19, 0, 99])
    assert lens.tolist() == [5, 20, 0, 0] and prompts.tolist() == [1, 9, 0, 0]
    assert tokens[0, :5].tolist() == [0, 1, 2, 77, 78]
    assert tokens[1, :20].tolist() == list(range(19)) + [5]
    h.append(3, 79)
    h.drop(3)                       # what was not uploaded yet goes, too
    h.put("new", [9] * 300, 300)    # takes its row, and needs more room
    tokens, lens, _ = h.rows(["new", 19])
    assert tokens[0, :300].tolist() == [9] * 300 and lens.tolist() == [300, 20]
    assert tokens[1, :20].tolist() == list(range(19)) + [5]
    h.put(19, [1, 2], 2)            # starts again
    assert h.rows([19])[1].tolist() == [2]
    assert tokens.dtype == torch.int32


def test_pack_mask():
    g = torch.Generator().manual_seed(1)
    for v in (1, 31, 32, 33, 997):
        a = torch.rand(3, v, generator=g) < 0.5
        bits = np.zeros((3, -(-v // 32) * 32), dtype=np.uint8)
        bits[:, :v] = a.numpy()
        want = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
        for dev in ("cpu", DEV):
            assert pack_mask(a.to(dev)).tolist() == want.tolist()
