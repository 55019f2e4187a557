#!/usr/bin/env python
"""Small fixed cases for profiler captures (one kernel, a few launches, ~1 GB on the device).

    python benchmarks/profile_case.py attn      # GQA decode, B=8, 16K tokens per sequence (537 MB of KV)
    python benchmarks/profile_case.py oproj     # o_proj, 8 tokens, K=8192, hidden 8192 (134 MB of W)
    python benchmarks/profile_case.py exchange  # fused exchange+combine, 4 ranks played by one launch
    python benchmarks/profile_case.py mla       # MLA fp8 decode, B=8, 16K tokens per sequence
    python benchmarks/profile_case.py mla_64k   # the same with 64K tokens per sequence (344 MB of cache, larger than L2)
    python benchmarks/profile_case.py fused     # one-kernel exchange+combine+o_proj, 8 ranks played by one launch
    python benchmarks/profile_case.py fused_rows  # the same with 64 tokens (slabs of a head group share the rows)
    python benchmarks/profile_case.py streamk   # stream-K o_proj, 8 tokens, K=8192, hidden 8192
    python benchmarks/profile_case.py combine   # stand-alone LSE combine, 8 ranks x 4096 rows x 512
    python benchmarks/profile_case.py tree      # tree attention, B=8, 16 drafted tokens each, 16K tokens per sequence (537 MB of KV)
    python benchmarks/profile_case.py tree_wide # the same for one sequence of 64K tokens and 64 drafted ones (268 MB of KV)
    python benchmarks/profile_case.py int4      # o_proj with 4-bit weights, 100 tokens, K=8192, hidden 8192
    python benchmarks/profile_case.py int4_few  # the same for 8 tokens
    python benchmarks/profile_case.py append    # 16384 rows of K and V into a paged cache, a quarter of them other ranks' (101 MB moved)
    python benchmarks/profile_case.py tables    # pages and slots of 64 prompts, 61000 tokens
"""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import torch  # noqa: E402


def main():
    which = sys.argv[1] if len(sys.argv) > 1 else "attn"
    launches = 3
    if which == "attn":
        from helix_a2a_b200.ops import attention
        B, ctx, Hq, Hkv, D, page = 8, 16384, 64, 8, 128, 16
        pages = B * ctx // page
        bt = torch.randperm(pages).int().view(B, -1).cuda()
        sl = torch.full((B,), ctx, dtype=torch.int32, device="cuda")
        kc = torch.randn(pages, Hkv, page, D, device="cuda", dtype=torch.bfloat16)
        vc = torch.randn(pages, Hkv, page, D, device="cuda", dtype=torch.bfloat16)
        q = torch.randn(B, Hq, D, device="cuda", dtype=torch.bfloat16)
        for _ in range(launches):
            attention.gqa_decode(q, kc, vc, bt, sl, max_seq_len=ctx)
    elif which == "oproj":
        from helix_a2a_b200.ops.oproj import oproj
        w = (torch.randn(8192, 8192, device="cuda") * 0.02).bfloat16()
        x = torch.randn(8, 8192, device="cuda").bfloat16()
        for _ in range(launches):
            oproj(x, w)
    elif which == "streamk":
        from helix_a2a_b200.ops.oproj import oproj
        w = (torch.randn(8192, 8192, device="cuda") * 0.02).bfloat16()
        x = torch.randn(8, 8192, device="cuda").bfloat16()
        for _ in range(launches):
            oproj(x, w, splits=-1)
    elif which == "append":
        from helix_a2a_b200.ops import paged
        qkv = torch.randn(16384, 3, 8, 128, device="cuda").half()
        kc, vc = (torch.zeros(1024, 32, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2))
        slots = torch.randperm(1024 * 32, device="cuda")[:16384]
        slots[torch.rand(16384, device="cuda") < 0.25] = -1
        for _ in range(launches):
            paged.append_kv(qkv[:, 1], qkv[:, 2], kc, vc, slots, layout="NHD")
    elif which == "tables":
        from helix_a2a_b200.ops import paged
        rows = 64 * 953

        def zeros(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device="cuda")

        free, starts = torch.randperm(64 * 64, device="cuda").int(), torch.arange(0, rows + 1, 953, device="cuda").int()
        for _ in range(launches):
            paged.extend_tables(zeros(64, 64), zeros(64), free, zeros(1), zeros(64), starts, rows=rows, page_size=16, mask_words=0)
    elif which in ("tree", "tree_wide"):
        from helix_a2a_b200.ops import attention, paged
        B, ctx, drafts = (8, 16384, 16) if which == "tree" else (1, 65536, 64)
        pages, words = ctx // 16 + drafts // 16, (drafts + 63) // 64

        def i32(*v):
            return torch.tensor(v, dtype=torch.int32, device="cuda")

        table = torch.randperm(B * pages).int().view(B, -1).cuda()
        plan = paged.extend_tables(table, i32(*[pages] * B), i32(), i32(0), i32(*[ctx] * B), i32(*range(0, B * drafts + 1, drafts)),
                                   rows=B * drafts, page_size=16, mask_words=words)
        kc, vc = (torch.randn(B * pages, 8, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        q = torch.randn(B * drafts, 64, 128, device="cuda", dtype=torch.bfloat16)
        for _ in range(launches):
            attention.tree_decode(q, kc, vc, table, plan.seq_lens, i32(*range(0, B * drafts + 1, drafts)), plan.draft_lens, plan.mask,
                                  max_seq_len=ctx + drafts, max_q_len=drafts)
    elif which in ("int4", "int4_few"):
        from helix_a2a_b200.ops import oproj
        few = which == "int4_few"
        w = oproj.quantize_weight_int4((torch.randn(8192, 8192, device="cuda") * 0.02).bfloat16(), zero_points=few)
        x = torch.randn(8 if few else 100, 8192, device="cuda").bfloat16()
        for _ in range(launches):
            oproj.oproj(x, w)
    elif which == "combine":
        import helix_a2a_b200 as helix
        o = torch.randn(8, 32, 128, 512, device="cuda").bfloat16()
        l = torch.randn(8, 32, 128, device="cuda")
        for _ in range(launches):
            helix.lse_combine(o, l)
    elif which in ("fused", "fused_rows"):
        import helix_a2a_b200 as helix
        from helix_a2a_b200.ops._ext import ops
        # per rank: K = 1024 in two head groups, 8 slabs; "fused_rows": 64 tokens, so the slabs share the rows
        cp, B, H, D, hidden = 8, (8 if which == "fused" else 64), 64, 128, 1024
        ws = helix.allocate_workspace(cp, 0)
        helix.init_workspace_all_rows(ws, cp)
        outs = torch.randn(cp, B, H, D, device="cuda").bfloat16()
        lses = torch.randn(cp, B, H, device="cuda")
        w = (torch.randn(cp, hidden, (H // cp) * D, device="cuda") * 0.05).bfloat16()
        for _ in range(launches):
            ops().alltoall_combine_oproj(outs, lses, w, ws, 0, cp, False, True, 0)
    elif which in ("mla", "mla_64k"):
        import math
        from helix_a2a_b200.ops import attention, reference_math as rm
        B, ctx, page = 8, (16384 if which == "mla" else 65536), 16
        pages = B * ctx // page
        bt = torch.randperm(pages).int().view(B, -1).cuda()
        sl = torch.full((B,), ctx, dtype=torch.int32, device="cuda")
        ckv, sc = rm.quantize_fp8_blockscaled(torch.randn(pages, page, 512, device="cuda"), 128)
        kpe = torch.randn(pages, page, 64, device="cuda").bfloat16()
        qn = (torch.randn(B, 128, 512, device="cuda") * 0.3).bfloat16()
        qp = (torch.randn(B, 128, 64, device="cuda") * 0.3).bfloat16()
        for _ in range(launches):
            attention.mla_decode(qn, qp, ckv, sc, kpe, bt, sl, scale=1 / math.sqrt(192), max_seq_len=ctx)
    else:
        import helix_a2a_b200 as helix
        from helix_a2a_b200.ops._ext import ops
        cp, B, H, D = 4, 64, 128, 512
        ws = helix.allocate_workspace(cp, 0)
        helix.init_workspace_all_rows(ws, cp)
        outs = torch.randn(cp, B, H, D, device="cuda").bfloat16()
        lses = torch.randn(cp, B, H, device="cuda")
        for _ in range(launches):
            ops().alltoall_combine(outs, lses, ws, 0, cp, 0, False, False, 0, True, 0, 0)
    torch.cuda.synchronize()
    print("done", which)


if __name__ == "__main__":
    main()
