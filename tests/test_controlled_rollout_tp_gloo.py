"""Controlled requests and top logprobs on a tensor-parallel engine (driver + follower replay) against one rank, gloo on
CPU: the driver alone controls and samples, and ends requests whose grammar allows nothing between the steps that the
follower replays."""

import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


class StopsAfter:
    """Allows multiples of three, and nothing after `stop` tokens."""

    def __init__(self, vocab, stop):
        self.vocab, self.stop = vocab, stop

    def fill_mask(self, output_tokens, words):
        from libra_b200.engine.rollout.controls import allow_tokens

        if len(output_tokens) < self.stop:
            allow_tokens(words, range(0, self.vocab, 3), self.vocab)


def _worker(rank, world, port, out_dir):
    import datetime

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=120))
    from libra_b200.engine.rollout.llm_engine import LLMEngine
    from libra_b200.engine.rollout.sampler import SamplingParams
    from libra_b200.models.qwen3 import ParamLayout, get_config, init_params, param_shapes
    from libra_b200.parallel.tensor_parallel import shard_full_params

    cfg = get_config("tiny")
    layout = ParamLayout(param_shapes(cfg))
    full = layout.views(torch.zeros(layout.numel))
    init_params(cfg, full, seed=3)
    full = {k: (v * 4 if v.dim() > 1 else v).clone() for k, v in full.items()}  # sharper logits
    local = shard_full_params(full, cfg, world, rank)
    eng = LLMEngine(cfg, local, kv_blocks=64, block_size=4, max_running=4, tp_group=dist.group.WORLD, tp_size=world,
                    tp_channel=dist.group.WORLD)
    if rank:
        eng.follower_loop()
    else:
        one = LLMEngine(cfg, full, kv_blocks=64, block_size=4, max_running=4)
        V = cfg.vocab_size
        prompts = [[5, 9, 13, 17, 21], [7, 7, 7], [100, 200, 300, 400, 500], [5, 9, 13, 17, 21], [1], [2, 3]]

        def params(i):
            kw = [dict(), dict(repetition_penalty=1.6, frequency_penalty=0.4, top_logprobs=5),
                  dict(grammar=StopsAfter(V, 2), top_logprobs=3), dict(allowed_token_ids=[3, 4, 5, 6], presence_penalty=2.0),
                  dict(grammar=StopsAfter(V, 0)), dict(logit_bias={11: 50.0}, top_logprobs=2)][i]
            return SamplingParams(max_tokens=6, temperature=0.0, **kw)

        for batch in ([0, 1, 2, 3, 4, 5], [4], [2, 4], [4, 4, 4], [1, 0]):  # (two of them end without a model step)
            got = eng.generate_sync([prompts[i] for i in batch], [params(i) for i in batch])
            want = one.generate_sync([prompts[i] for i in batch], [params(i) for i in batch])
            for g, w in zip(got, want):
                assert (g.output_tokens, g.finish_reason) == (w.output_tokens, w.finish_reason)
                assert [[t for t, _ in row] for row in g.output_top_logprobs] == \
                    [[t for t, _ in row] for row in w.output_top_logprobs]
                assert all(abs(a - b) < 1e-3 for a, b in zip(g.output_logprobs, w.output_logprobs))
            assert eng.kv.seqs == {} and not eng._controls._row
        eng.shutdown()
    assert eng.kv.seqs == {}, "the follower replayed every release"
    open(os.path.join(out_dir, f"ok_{rank}"), "w").close()
    dist.destroy_process_group()


def test_controlled_tp_rollout_matches_single_rank(tmp_path):
    mp.start_processes(_worker, args=(2, _port(), str(tmp_path)), nprocs=2, join=True, start_method="spawn")
    assert {p.name for p in tmp_path.iterdir()} == {"ok_0", "ok_1"}
