# GPU box: what each part of the range coder's loop costs - the generated loop with parts left out (timing only: results of the
# variants are wrong by construction), through tools/ubench_chain_f64.hip
set -e
cd /root/repo
for v in "product:" "no_checkpoints:GZ_GEN_CKPT=0" "no_hop:GZ_GEN_HOP=0" "no_prep:GZ_GEN_PREP=0" "bare:GZ_GEN_HOP=0 GZ_GEN_CKPT=0 GZ_GEN_PREP=0" "bare_operands_do_not_rotate:GZ_GEN_NOROT=1 GZ_GEN_HOP=0 GZ_GEN_CKPT=0 GZ_GEN_PREP=0" "constant_one:GZ_GEN_ONE=1" "loads_spread:GZ_GEN_SPREAD=8" "bare_loads_spread:GZ_GEN_SPREAD=8 GZ_GEN_HOP=0 GZ_GEN_CKPT=0 GZ_GEN_PREP=0"; do
    name=${v%%:*}; envs=${v#*:}
    env $envs python tools/gen_chain_asm.py /tmp/chain_$name.h
    hipcc -O3 --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -ffp-contract=off -I tools -DGZ_CHAIN_HDR="\"/tmp/chain_$name.h\"" tools/ubench_chain_f64.hip -o /tmp/ub_$name 2>/dev/null
    echo "== $name"
    timeout 120 /tmp/ub_$name 2>&1 | grep "hop:  1 chains\|exactness \[hop" | grep "hop:  1 chains\|exactness \[hop" | head -3
done
