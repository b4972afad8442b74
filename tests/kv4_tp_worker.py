"""Worker of the test of 4-bit pages under tensor parallelism (launched with torch.distributed.run over gloo): greedy tokens of two prompts, written by rank 0."""
import json
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch
import torch.distributed as dist


def main():
    dist.init_process_group("gloo")
    from flyingfish_b200.api import Model
    from flyingfish_b200.config import Settings
    from flyingfish_b200.parallel.comm import TPComm
    comm = TPComm.create(dist.group.WORLD, torch.device("cpu"), slot_bytes=8 << 20)
    m = Model.load("tiny-llama", Settings(capacity=256, max_batch=4, graph=False, kv_format="affine4"), device="cpu", seed=0, comm=comm)
    tokens = m.generate_batch(json.loads(Path(sys.argv[1]).read_text()), 8)
    page = list(m.engine.kv.k[0].shape)
    dist.barrier()
    if dist.get_rank() == 0:
        Path(sys.argv[2]).write_text(json.dumps({"tokens": tokens, "page": page}))
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
