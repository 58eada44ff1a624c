"""`generate_shared` of a tensor-parallel model in a group of one rank: NCCL, the pushed and the one-shot all-reduce, each in a captured step, and changes
between them.  The child reports its exceptions."""
import datetime
import os
import sys
import traceback

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def _worker(port, q):
    try:
        sys.path.insert(0, ROOT)
        sys.path.insert(0, os.path.join(ROOT, "sbvr-cpu-arm_b200"))
        os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
        os.environ["NCCL_NVLS_ENABLE"] = "0"
        os.environ["TORCH_SYMM_MEM_DISABLE_MULTICAST"] = "1"
        import torch.distributed as dist
        from models.sbvr_llama import LlamaConfig, SBVRLlamaForCausalLM
        torch.cuda.set_device(0)
        dev = torch.device("cuda", 0)
        dist.init_process_group("nccl", rank=0, world_size=1, device_id=dev, timeout=datetime.timedelta(seconds=90))
        cfg = LlamaConfig.preset("tiny8")
        m = SBVRLlamaForCausalLM(cfg, device=dev, tp_group=dist.group.WORLD, max_batch=3, max_ctx=64).init_synthetic(3)
        m.attach_pages(40, 16, max_seqs=3)
        g = torch.Generator(device=dev).manual_seed(9)
        prefix = torch.randint(0, cfg.vocab_size, (37,), device=dev, generator=g)
        prompts = torch.randint(0, cfg.vocab_size, (3, 7), device=dev, generator=g)
        said = []

        def both(what):
            eager = m.generate_shared(prefix, prompts, 6, prompt_lengths=[7, 1, 4], use_graph=False)
            said.append((what, bool(torch.equal(eager, m.generate_shared(prefix, prompts, 6, prompt_lengths=[7, 1, 4])))))
        both("NCCL")
        if m.enable_fused_allreduce(16):
            both("pushed")
            m.set_pushed_allreduce(False)
            both("one-shot")
            m.set_pushed_allreduce(True)
            m.enable_fused_allreduce(16)
            both("pushed, another block")
        m._drop_graphs()                           # (before the group that their collectives belong to)
        q.put(("ok", said))
        dist.destroy_process_group()
    except Exception:
        q.put(("error", traceback.format_exc()))


def test_generate_shared_in_a_group_of_one():
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_worker, args=(29500 + (os.getpid() + 61) % 2000, q))
    p.start()
    try:
        status, said = q.get(timeout=240)
    finally:
        p.join(150)
        if p.is_alive():
            p.terminate()
    assert status == "ok", said
    assert said and all(same for _, same in said), said
