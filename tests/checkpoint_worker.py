"""Worker of the multi-rank training test (launched by torch.distributed.run, gloo, the ranks may share one GPU): one
training step of DistSAGE per exchange mode with 8-bit checkpoints and with the loss of many classes in pieces, against the
plain step on the same partition."""
import os
import sys

import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def main():
    os.environ["SGNN_DIST_BACKEND"] = "gloo"
    from super_gnn_b200 import graphsage, synthetic
    from super_gnn_b200.communicator import Communicator
    from super_gnn_b200.data_manager import build_distributed_graph, build_distributed_graph_pre_post, partition_edges
    from super_gnn_b200.quantizer import Quantizer_for_all_procs

    Communicator(32, is_async=True)
    rank, W = Communicator.ctx.init_dist_group()
    device = torch.device("cuda", torch.cuda.current_device())
    n, fin, hid, ncls = 2400, 48, 64, 20
    s, t = synthetic.rmat_edges(n, 24_000, 0.57, 0.19, 0.19, 0.05, seed=7)
    s, t = synthetic.symmetrize_dedup(s, t, n)
    s, t = synthetic.random_relabel(s, t, n, seed=7)
    begins = synthetic.even_ranges(n, W)
    local_edges, remote_edges = partition_edges(s, t, begins, rank)
    gen = torch.Generator().manual_seed(3)
    x_all, labels = torch.randn(n, fin, generator=gen), torch.randint(0, ncls, (n,), generator=gen)
    train = torch.rand(n, generator=gen) < 0.4
    masks = [(torch.rand(n, hid, generator=gen) >= 0.5).float() * 2 for _ in range(2)]
    lo, hi = begins[rank], begins[rank + 1]
    failures = []
    for is_pre in (False, True):
        for bits in (32, 2):
            Communicator.ctx.num_bits = bits
            Quantizer_for_all_procs(W, bits)
            build = build_distributed_graph_pre_post if is_pre else build_distributed_graph
            graph = build(local_edges, remote_edges, begins, hid, bits, device=device)
            for fold in (True, False):
                graph.set_fold_mean(fold)
                results = {}
                for name, extra in (("plain", {}), ("kept in 8 bits", dict(checkpoint_bits=8)), ("in pieces", dict(chunked_loss=True)),
                                    ("both", dict(checkpoint_bits=8, chunked_loss=True))):
                    torch.manual_seed(0)
                    model, _ = graphsage.create_model_and_optimizer(
                        dict(in_channels=fin, hidden_channels=hid, out_channels=ncls, num_layers=3, dropout=0.5, num_bits=bits,
                             is_pre_delay=is_pre, **extra), device=device)
                    core = model.module
                    core.dropout_masks = [m[lo:hi].to(device) for m in masks]
                    core.project_first = False  # the reference's place of the exchange in all of them
                    model.train()
                    x, lab, m = x_all[lo:hi].to(device), labels[lo:hi].to(device), train[lo:hi].to(device)
                    if core.can_fuse_loss(x, graph):
                        loss = model(graph, x, lab, None, loss_mask=m, loss_inv_count=1.0 / float(train.sum()), loss_unit_grad=True)
                    else:
                        out = model(graph, x)
                        loss = torch.nn.functional.nll_loss(out[m], lab[m], reduction="sum") / float(train.sum())
                    loss.backward()
                    total = loss.detach().clone()
                    dist.all_reduce(total)
                    results[name] = (float(total), {k: v.grad.detach().clone() for k, v in core.named_parameters()})
                want_loss, want = results["plain"]
                for name, (value, grads) in results.items():
                    tag = f"{name}, pre={is_pre} bits={bits} fold={fold}"
                    # two fp32 computations of the same forward; with 2 bits a code next to a border may turn
                    if abs(value - want_loss) > (1e-5 if bits == 32 else 1e-3) * abs(want_loss):
                        failures.append(f"{tag}: loss {value} vs {want_loss}")
                    for k, g in want.items():
                        off, size = float((grads[k] - g).norm()), float(g.norm())
                        # activations off by half a step of 255 (and signs of units next to the relu's corner), else fp32
                        # rounding; 2-bit gradient rows are quantised again, so what differs before differs by a step there
                        bound = 0.15 if "8" in name or name == "both" or bits == 2 else 1e-4
                        if not off <= bound * size:
                            failures.append(f"{tag}: gradient of {k} off by {off:.3e} of {size:.3e}")
    everyone = [None] * W
    dist.all_gather_object(everyone, failures)
    dist.destroy_process_group()
    if any(everyone):
        print("\n".join(sorted({f for fs in everyone for f in fs})[:20]), flush=True)
        sys.exit(1)


if __name__ == "__main__":
    main()
