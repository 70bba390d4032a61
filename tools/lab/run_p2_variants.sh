#!/bin/bash
# Lab (GPU box): time every tools/lab/p2_<name> on the ViT shape (kernel id 14) and bit-compare with kernel 11.
R=$GRAFT_REPO_ROOT
for name in "$@"; do
  echo "=== $name"
  for rep in 1 2; do LAB_CMP=11 $R/tools/lab/p2_$name 14 2>/dev/null | grep -E "^kernel|different BITS"; done
done
