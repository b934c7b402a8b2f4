// One (element type, cache code) instantiation of the tree attention per object file: compiled with
// -DSPFA_TREE_T={spfa::f16,spfa::bf16} -DSPFA_TREE_CODE={0,1,2}.
#include "spfa_tree.hpp"
